"""8-bit block cache: keys and values in 8 bits with one fp32 scale for each page, head and side, for the tokens that
are not held in spherical pages (the newest of a sequence, a prompt that is not encoded yet).  Attention over it and
over a PagedCache merge by log-sum-exp: give both decodes an `out_partial` and join them with merge_partials.

    cache = new_block_cache(n_pages, Hkv, 16, 128, block_table)       # torch.int8, or torch.float8_e4m3fn
    cache.seq_lens += 1                                               # the step's token counts as held
    append_blocks(cache, k, v)                                        # k, v [B, 1, Hkv, dh], keys post-RoPE
    out = decode_blocks(q, cache)                                     # q [B, Hq, dh]

Every call is about the last n_b tokens of each sequence b, positions seq_lens[b] - n_b .. seq_lens[b] - 1: the same n for
all (a dense [B, n, ...] tensor), or rows cu[b] .. cu[b + 1] - 1 of a [rows, ...] tensor (cu: int32 [B + 1] on the device;
rows before cu[0] and from cu[B] on are padding and left alone).  Lengths live on the device and no call reads them back, so all of them record
into CUDA graphs.  Sequences whose numbers do not fit and bad table entries raise bits of `cache.status`
(ops.check_status reads it).  Calls run on the current stream of the cache's device; their workspaces come from torch's
allocator per call, so calls on several streams do not meet in them.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib

try:
    from torch._C import _cuda_getCurrentRawStream, _cuda_getDevice
except ImportError:  # a torch without CUDA: every call is refused before these are needed
    _cuda_getCurrentRawStream, _cuda_getDevice = None, lambda: -1

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_STORE = {torch.int8: _lib.BLOCKS_I8, torch.float8_e4m3fn: _lib.BLOCKS_E4M3}


@dataclass
class BlockCache:
    """Device-resident 8-bit cache of one attention layer.  A value is code * scale; codes of a sequence's tokens are finite (append_blocks
    writes no others: a token without a finite value is a scale that is not finite)."""
    k_codes: torch.Tensor      # i8 | float8_e4m3fn [n_pages, Hkv, page_size, dh]
    v_codes: torch.Tensor      # the same
    k_scale: torch.Tensor      # f32 [n_pages, Hkv]
    v_scale: torch.Tensor      # f32 [n_pages, Hkv]
    block_table: torch.Tensor  # i32 [B, max_blocks]: page of tokens page_size * i ..; entries past a sequence's end, or before the
                               # page of the `first` that a call is given: anything
    seq_lens: torch.Tensor     # i32 [B]: tokens held, those of the present step among them
    status: Optional[torch.Tensor] = None

    def __post_init__(self):
        if self.status is None and self.k_codes.is_cuda:
            self.status = torch.zeros(1, dtype=torch.int32, device=self.k_codes.device)

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]

    @property
    def dh(self) -> int:
        return self.k_codes.shape[3]

    @property
    def Hkv(self) -> int:
        return self.k_codes.shape[1]


def new_block_cache(n_pages: int, Hkv: int, page_size: int, dh: int, block_table: torch.Tensor,
                    store: torch.dtype = torch.int8) -> BlockCache:
    """An empty cache on block_table's device."""
    if store not in _STORE:
        raise ValueError(f"store {store}: torch.int8 or torch.float8_e4m3fn")
    if page_size not in (16, 32, 64, 128) or dh not in (64, 128):
        raise ValueError(f"page_size={page_size} (16, 32, 64, 128), dh={dh} (64, 128)")
    dev = block_table.device
    codes = [torch.zeros(n_pages, Hkv, page_size, dh, dtype=torch.int8, device=dev).view(store) for _ in range(2)]
    scales = [torch.zeros(n_pages, Hkv, dtype=torch.float32, device=dev) for _ in range(2)]
    return BlockCache(*codes, *scales, block_table, torch.zeros(block_table.shape[0], dtype=torch.int32, device=dev))


_calls = None  # (host function, addresses of the library's functions) of each operator


def _bind() -> dict:
    global _calls
    lib, host = _lib.load(), _lib.host_tables()

    def at(name: str) -> int:
        return C.cast(getattr(lib, name), C.c_void_p).value
    last = at("sphkv_last_error")
    _calls = {name: (getattr(host, "blocks_" + name), at("sphkv_blocks_" + name), last) for name in ("append", "read", "decode", "attend")}
    _calls["scratch"] = (at("sphkv_blocks_decode_scratch_bytes"), at("sphkv_blocks_attend_scratch_bytes"))
    return _calls


def _call(name: str, cache: BlockCache, ends: Optional[torch.Tensor], *args):
    """The host module checks the arguments, makes outputs and workspaces and calls the library, on the current stream of the
    cache's device; a text is its reason to refuse."""
    host, fn, last = (_calls or _bind())[name]
    k = cache.k_codes
    dev = k.get_device()
    if dev < 0:
        raise _lib.SphKVError("block cache: expected contiguous CUDA tensors on one device")
    here = _cuda_getDevice()
    if dev != here:
        torch._C._cuda_setDevice(dev)
    try:
        r = host(fn, last, _cuda_getCurrentRawStream(dev), k, cache.v_codes, cache.k_scale, cache.v_scale, cache.block_table, ends,
                 cache.status, *args)
    finally:
        if dev != here:
            torch._C._cuda_setDevice(here)
    if type(r) is str:
        raise _lib.SphKVError(r)
    return r


def _type(dtype: Optional[torch.dtype]) -> int:
    if dtype is None:
        return -1
    if dtype not in _DT:
        raise _lib.SphKVError("out_dtype: float32, bfloat16 or float16")
    return _DT[dtype]


def append_blocks(cache: BlockCache, k: torch.Tensor, v: torch.Tensor, cu_new: Optional[torch.Tensor] = None) -> None:
    """Quantises the last n_b tokens of every sequence into its pages.

    k, v: [B, n, Hkv, dh], or [rows, Hkv, dh] with cu_new; f32, bf16 or f16, elements of a head contiguous, rows of all sequences
    one stride apart, other strides as they come (slices of a fused projection).  seq_lens counts the new tokens already.  A page keeps one scale per head and
    side, max |x| / 127 (e4m3: / 448) of all it was given: where new tokens raise it, the page's earlier tokens of the sequence are
    re-quantised.  Codes are the nearest to x / scale, ties to even.  An infinity or NaN makes its page, head and side read
    back as NaN.  A page that is appended to belongs to one sequence, and stands once in its row of the table."""
    _call("append", cache, cache.seq_lens, k, v, cu_new)


def read_blocks(cache: BlockCache, n: Optional[int] = None, cu_rows: Optional[torch.Tensor] = None, rows: Optional[int] = None,
                ends: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = torch.float32,
                out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of a run of tokens of every sequence as dense rows: the last `n` (-> [B, n, Hkv, dh]), or cu_rows[b + 1]
    - cu_rows[b] of them (-> [rows, Hkv, dh], `rows` the host's bound of cu_rows[B]).  `ends` (int32 [B]) takes the tokens
    before position ends[b] instead of before seq_lens[b].  The rows have the layout that encode_pages takes, and the keys are what
    was appended: post-RoPE ones make pages that are decoded with decode_paged(rope=None); a decode with a RoPE table expects pages
    of pre-RoPE keys."""
    if (n is None) == (cu_rows is None):
        raise _lib.SphKVError("read_blocks: either n, or cu_rows with rows")
    k, v = out if out is not None else (None, None)
    if cu_rows is not None and rows is None:
        if out is None:
            raise _lib.SphKVError("read_blocks: cu_rows needs rows")
        rows = k.shape[0]
    return _call("read", cache, cache.seq_lens if ends is None else ends, -1 if n is None else n, cu_rows, 0 if rows is None else rows,
                 _type(torch.float32 if out_dtype is None else out_dtype), k, v)


def decode_blocks(q: torch.Tensor, cache: BlockCache, first: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                  out_partial: Optional[torch.Tensor] = None, want_out: bool = True) -> Optional[torch.Tensor]:
    """Attention of one query a sequence, q [B, Hq, dh] (f32, bf16, f16), over its tokens first[b] .. seq_lens[b] - 1 (first:
    int32 [B], None = 0).  Returns [B, Hq, dh]; zeros where a sequence has no such token.  `out_partial` (f32 [B, Hq, dh + 2])
    receives (max, sum, acc), un-normalised, as decode_paged writes them.  sm_scale: any finite number, None = 1 / sqrt(dh).  Errors are
    those of fp32 sums, whatever scales stand beside one another."""
    return _call("decode", cache, cache.seq_lens, (_calls or _bind())["scratch"][0], q, first, sm_scale,
                 _type(out_dtype), out, out_partial, want_out)


def attend_blocks(q: torch.Tensor, cache: BlockCache, cu_new: Optional[torch.Tensor] = None, first: Optional[torch.Tensor] = None,
                  sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                  out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Causal attention of the last n_b tokens of every sequence (appended before): the query at position p sees tokens
    first[b] .. p.  q [B, n, Hq, dh], or [rows, Hq, dh] with cu_new (rows one stride apart, as append_blocks takes them); bf16 or f16.
    Returns q's shape; zeros where a query sees nothing, and padding rows are not written.  sm_scale as for decode_blocks.  Softmax
    weights are rounded once to f16 (11 bits), with fp32 outputs too, and values below 2^-80 of the sequence's largest value scale count as
    zeros; calls of up to 8 / (Hq / Hkv) tokens a sequence have decode_blocks' errors."""
    return _call("attend", cache, cache.seq_lens, (_calls or _bind())["scratch"][1], q, cu_new, first,
                 sm_scale, _type(out_dtype), out)
