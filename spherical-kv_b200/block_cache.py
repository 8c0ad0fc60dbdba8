"""8-bit block cache: keys and values in 8 bits with one fp32 scale for each page, head and side, for the tokens that
are not held in spherical pages (the newest of a sequence, a prompt that is not encoded yet).  Attention over it and
over a PagedCache merge by log-sum-exp: give both decodes an `out_partial` and join them with merge_partials.

    cache = new_block_cache(n_pages, Hkv, 16, 128, block_table)       # torch.int8, or torch.float8_e4m3fn
    cache.seq_lens += 1                                               # the step's token counts as held
    append_blocks(cache, k, v)                                        # k, v [B, 1, Hkv, dh], keys post-RoPE
    out = decode_blocks(q, cache)                                     # q [B, Hq, dh]

Every call is about the last n_b tokens of each sequence b, positions seq_lens[b] - n_b .. seq_lens[b] - 1: the same n for
all (a dense [B, n, ...] tensor), or rows cu[b] .. cu[b + 1] - 1 of a [rows, ...] tensor (cu: int32 [B + 1] on the device;
rows from cu[B] on are padding and left alone).  Lengths live on the device and no call reads them back, so all of them record
into CUDA graphs.  Sequences whose numbers do not fit and bad table entries raise bits of `cache.status`
(ops.check_status reads it).  Calls run on the current stream of the cache's device; their workspaces come from torch's
allocator per call, so calls on several streams do not meet in them.
"""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Optional, Tuple

import torch

from . import _lib

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_STORE = {torch.int8: _lib.BLOCKS_I8, torch.float8_e4m3fn: _lib.BLOCKS_E4M3}


@dataclass
class BlockCache:
    """Device-resident 8-bit cache of one attention layer.  A value is code * scale."""
    k_codes: torch.Tensor      # i8 | float8_e4m3fn [n_pages, Hkv, page_size, dh]
    v_codes: torch.Tensor      # the same
    k_scale: torch.Tensor      # f32 [n_pages, Hkv]
    v_scale: torch.Tensor      # f32 [n_pages, Hkv]
    block_table: torch.Tensor  # i32 [B, max_blocks]: page of tokens page_size * i ..; entries past a sequence's end: anything
    seq_lens: torch.Tensor     # i32 [B]: tokens held, those of the present step among them
    status: Optional[torch.Tensor] = None
    extra: dict = field(default_factory=dict)

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


def _err(text: str):
    raise _lib.SphKVError(text)


def _i32(t: Optional[torch.Tensor], n: int, dev: torch.device, name: str) -> int:
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.device != dev or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        _err(f"{name}: expected a contiguous int32 tensor of {n} on {dev}")
    return t.data_ptr()


def _view(cache: BlockCache, ends: Optional[torch.Tensor] = None) -> Tuple[bytes, torch.device, int, int, int, int]:
    """The cache as the library's struct (packed), its device, B, Hkv, page size and head dim."""
    kc, vc, ks, vs, bt = cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, cache.block_table
    dev, dt, shape = kc.device, kc.dtype, kc.shape
    if dt not in _STORE or len(shape) != 4 or vc.dtype != dt or vc.shape != shape:
        _err("block cache: codes are int8 or float8_e4m3fn [n_pages, Hkv, page_size, dh], the same for keys and values")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32 or ks.shape != shape[:2] or vs.shape != shape[:2]:
        _err("block cache: scales are float32 [n_pages, Hkv]")
    if bt.dtype != torch.int32 or bt.dim() != 2:
        _err("block cache: block_table is int32 [B, max_blocks]")
    st = cache.status
    if st is not None and (st.dtype != torch.int32 or st.device != dev):
        _err("block cache: status is int32 on the cache's device")
    for t in (kc, vc, ks, vs, bt):
        if not t.is_cuda or t.device != dev or not t.is_contiguous():
            _err("block cache: expected contiguous CUDA tensors on one device")
    B, most = bt.shape
    ends_at = _i32(cache.seq_lens if ends is None else ends, B, dev, "seq_lens" if ends is None else "ends")
    n_pages, hkv, page, dh = shape
    return (_lib.Blocks.packer.pack(kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), bt.data_ptr(), ends_at,
                                    0 if st is None else st.data_ptr(), n_pages, hkv, page, dh, B, most, _STORE[dt]), dev, B, hkv, page, dh)


class _on:
    """The device made current, only where it is not."""
    __slots__ = ("index", "before")

    def __init__(self, dev: torch.device):
        self.index = dev.index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch._C._cuda_setDevice(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch._C._cuda_setDevice(self.before)


def _dense(t: torch.Tensor, cu: Optional[torch.Tensor], B: int, heads: Optional[int], dh: int, dev: torch.device, name: str):
    """Rows, heads, row and head stride of [B, n, heads, dh] (cu None) or [rows, heads, dh]."""
    if t.device != dev or t.dtype not in _DT:
        _err(f"{name}: expected float32, bfloat16 or float16 on {dev}")
    shape, stride = t.shape, t.stride()
    want = 4 if cu is None else 3
    if len(shape) != want or shape[-1] != dh or (heads is not None and shape[-2] != heads) or (cu is None and shape[0] != B):
        _err(f"{name}: shape {tuple(shape)}, expected " +
             (f"[{B}, n, {heads or 'Hq'}, {dh}]" if cu is None else f"[rows, {heads or 'Hq'}, {dh}] with cu_new"))
    if dh > 1 and stride[-1] != 1:
        _err(f"{name}: elements of a head must be contiguous")
    rows = shape[0] * shape[1] if cu is None else shape[0]
    if cu is None and shape[0] > 1 and shape[1] > 1 and stride[0] != shape[1] * stride[1]:
        _err(f"{name}: rows of all sequences must be one stride apart")
    row = stride[1] if cu is None and shape[1] > 1 else stride[0]
    return rows, shape[-2], row, stride[-2]


def append_blocks(cache: BlockCache, k: torch.Tensor, v: torch.Tensor, cu_new: Optional[torch.Tensor] = None) -> None:
    """Quantises the last n_b tokens of every sequence into its pages.

    k, v: [B, n, Hkv, dh], or [rows, Hkv, dh] with cu_new; f32, bf16 or f16, elements of a head contiguous, other strides as
    they come (slices of a fused projection).  seq_lens counts the new tokens already.  A page keeps one scale per head and
    side, max |x| / 127 (e4m3: / 448) of all it was given: where new tokens raise it, the page's earlier tokens of the sequence are
    re-quantised.  Codes are the nearest to x / scale, ties to even.  An infinity or NaN makes its page, head and side read
    back as NaN.  Two sequences must not append to the same page."""
    lib = _lib.load()
    view, dev, B, hkv, _, dh = _view(cache)
    rows, _, k_row, k_head = _dense(k, cu_new, B, hkv, dh, dev, "k")
    if v.shape != k.shape or v.dtype != k.dtype:
        _err("v: expected k's shape and type")
    _, _, v_row, v_head = _dense(v, cu_new, B, hkv, dh, dev, "v")
    with _on(dev):
        _lib.check(lib.sphkv_blocks_append(view, k.data_ptr(), v.data_ptr(), _DT[k.dtype], k_row, k_head, v_row, v_head,
                                           _i32(cu_new, B + 1, dev, "cu_new"), rows, _lib.stream_ptr()), "sphkv_blocks_append")


def read_blocks(cache: BlockCache, n: Optional[int] = None, cu_rows: Optional[torch.Tensor] = None, rows: Optional[int] = None,
                ends: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32,
                out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of a run of tokens of every sequence as dense rows: the last `n` (-> [B, n, Hkv, dh]), or cu_rows[b + 1]
    - cu_rows[b] of them (-> [rows, Hkv, dh], `rows` the host's bound of cu_rows[B]).  `ends` (int32 [B]) takes the tokens
    before position ends[b] instead of before seq_lens[b]: encode_pages can take them as they come out."""
    lib = _lib.load()
    view, dev, B, hkv, _, dh = _view(cache, ends)
    if (n is None) == (cu_rows is None):
        _err("read_blocks: either n, or cu_rows with rows")
    if cu_rows is None:
        rows, shape = B * n, (B, n, hkv, dh)
    else:
        if rows is None:
            rows = out[0].shape[0] if out is not None else _err("read_blocks: cu_rows needs rows")
        shape = (rows, hkv, dh)
    if out is None:
        if out_dtype not in _DT:
            _err("read_blocks: out_dtype float32, bfloat16 or float16")
        out = (torch.empty(shape, dtype=out_dtype, device=dev), torch.empty(shape, dtype=out_dtype, device=dev))
    k, v = out
    for t in out:
        if t.shape != shape or t.dtype not in _DT or t.dtype != k.dtype or t.device != dev or not t.is_contiguous():
            _err(f"out: expected two contiguous tensors {shape} of one type on {dev}")
    with _on(dev):
        _lib.check(lib.sphkv_blocks_read(view, k.data_ptr(), v.data_ptr(), _DT[k.dtype], _i32(cu_rows, B + 1, dev, "cu_rows"), rows,
                                         _lib.stream_ptr()), "sphkv_blocks_read")
    return k, v


def _output(out: Optional[torch.Tensor], shape, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    if out is None:
        if dtype not in _DT:
            _err("out_dtype: float32, bfloat16 or float16")
        return torch.empty(shape, dtype=dtype, device=dev)
    if out.shape != shape or out.dtype not in _DT or out.device != dev or not out.is_contiguous():
        _err(f"out: expected a contiguous tensor {tuple(shape)} on {dev}")
    return out


def decode_blocks(q: torch.Tensor, cache: BlockCache, first: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                  out_partial: Optional[torch.Tensor] = None, want_out: bool = True) -> Optional[torch.Tensor]:
    """Attention of one query a sequence, q [B, Hq, dh] (f32, bf16, f16), over its tokens first[b] .. seq_lens[b] - 1 (first:
    int32 [B], None = 0).  Returns [B, Hq, dh]; zeros where a sequence has no such token.  `out_partial` (f32 [B, Hq, dh + 2])
    receives (max, sum, acc), un-normalised, as decode_paged writes them."""
    lib = _lib.load()
    view, dev, B, hkv, _, dh = _view(cache)
    if q.device != dev or q.dtype not in _DT or q.dim() != 3 or q.shape[0] != B or q.shape[2] != dh or q.stride(2) != 1:
        _err(f"q: expected [{B}, Hq, {dh}] of float32, bfloat16 or float16 on {dev}, elements of a head contiguous")
    Hq = q.shape[1]
    if out is not None or want_out:
        out = _output(out, q.shape, out_dtype or q.dtype, dev)
    if out_partial is not None and (out_partial.dtype != torch.float32 or out_partial.device != dev or not out_partial.is_contiguous()
                                    or out_partial.shape != (B, Hq, dh + 2)):
        _err(f"out_partial: expected contiguous float32 [{B}, {Hq}, {dh + 2}] on {dev}")
    with _on(dev):
        need = lib.sphkv_blocks_decode_scratch_bytes(B, Hq, hkv, dh)
        if need < 0:
            _err(f"decode_blocks: Hq={Hq}, Hkv={hkv}, dh={dh} rejected (at most {_lib.MAX_GQA} query heads per KV head)")
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(lib.sphkv_blocks_decode(view, q.data_ptr(), _DT[q.dtype], q.stride(0), q.stride(1), _i32(first, B, dev, "first"),
                                           0 if out is None else out.data_ptr(), 0 if out is None else _DT[out.dtype],
                                           0 if out_partial is None else out_partial.data_ptr(), scratch.data_ptr(), need, Hq,
                                           1.0 / math.sqrt(dh) if sm_scale is None else sm_scale, _lib.stream_ptr()),
                   "sphkv_blocks_decode")
    return out


def attend_blocks(q: torch.Tensor, cache: BlockCache, cu_new: Optional[torch.Tensor] = None, first: Optional[torch.Tensor] = None,
                  sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                  out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Causal attention of the last n_b tokens of every sequence (appended before): the query at position p sees tokens
    first[b] .. p.  q [B, n, Hq, dh], or [rows, Hq, dh] with cu_new; bf16 or f16.  Returns q's shape; zeros where a query sees
    nothing, and padding rows are not written."""
    lib = _lib.load()
    view, dev, B, hkv, _, dh = _view(cache)
    rows, Hq, row, head = _dense(q, cu_new, B, None, dh, dev, "q")
    if q.dtype == torch.float32:
        _err("attend_blocks: q is bfloat16 or float16")
    out = _output(out, q.shape, out_dtype or q.dtype, dev)
    with _on(dev):
        need = lib.sphkv_blocks_attend_scratch_bytes(B, rows, Hq, hkv, dh)
        if need < 0:
            _err(f"attend_blocks: Hq={Hq}, Hkv={hkv}, dh={dh} rejected (at most {_lib.MAX_GQA} query heads per KV head)")
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(lib.sphkv_blocks_attend(view, q.data_ptr(), _DT[q.dtype], row, head, _i32(cu_new, B + 1, dev, "cu_new"), rows,
                                           _i32(first, B, dev, "first"), out.data_ptr(), _DT[out.dtype], scratch.data_ptr(), need, Hq,
                                           1.0 / math.sqrt(dh) if sm_scale is None else sm_scale, _lib.stream_ptr()),
                   "sphkv_blocks_attend")
    return out
