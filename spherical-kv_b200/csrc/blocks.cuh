// What the kernels of the 8-bit block cache share: which tokens a piece of work is about, and 8-bit codes to and from floats.
#pragma once
#include "tcgen05.cuh"

namespace sphkv {

// A call's dense rows: `rows` of them, cut into sequences by cu, or evenly where cu is NULL.
struct BlockRows {
  const int32_t* cu;
  int32_t rows, even;  // even: rows / B
  int32_t mul;         // rows are dealt in units of 1 / mul of a dense row (a query row for each head of a group)
  bool lone;           // one row a sequence that need not be among its tokens: a sequence may be empty
};

// Work on the n_b tokens of every sequence is dealt in pieces (pages that they touch; groups of queries) through a fixed
// number of slots that the host can tell without reading cu: a sequence has at most (n_b >> shift) + extra pieces, and
// its slots start at (cu[b] >> shift) + extra * b, which leaves room for (n_b >> shift) + extra of them.
__host__ __device__ inline int block_slots_even(int n, int shift, int extra) {  // of one sequence
  return n <= 0 ? 0 : ((n + (1 << shift) - 1) >> shift) + extra - 1;
}
inline int64_t block_slots(const BlockRows& r, int B, int shift, int extra) {
  if (r.cu == nullptr) return (int64_t)B * block_slots_even(r.even * r.mul, shift, extra);
  return ((int64_t)r.rows * r.mul >> shift) + (int64_t)extra * B;
}

struct BlockPiece {
  int b, j;     // sequence, and the piece's number in it; b < 0: no such sequence
  int row0, n;  // the sequence's dense rows
  int end;      // its tokens; negative: they do not fit, and the status word says so
};
__device__ __forceinline__ void bad_status(const sphkv_blocks& c, int bit) {
  if (c.status) atomicOr(c.status, bit);
}
__device__ __forceinline__ bool bad_rows(const BlockRows& r, int lo, int hi) { return lo < 0 || hi < lo || hi > r.rows; }
__device__ __forceinline__ BlockPiece checked_piece(const sphkv_blocks& c, const BlockRows& r, int b, int j, int lo, int hi, int end) {
  BlockPiece p = {b, j, lo, hi - lo, end};
  if (b < 0 || j < 0 || bad_rows(r, lo, hi)) {  // j < 0: a slot of rows before cu[0], which are no sequence's
    p.b = -1;
    p.n = 0;
    return p;
  }
  if (p.end < 0 || p.end > (int64_t)c.max_blocks * c.page_size || (p.n > p.end && !r.lone)) {
    bad_status(c, SPHKV_ST_BAD_LENGTH);
    p.end = -1;
  }
  return p;
}
__device__ __forceinline__ BlockPiece even_piece(const sphkv_blocks& c, const BlockRows& r, int slot, int shift, int extra) {
  const int per = block_slots_even(r.even * r.mul, shift, extra), b = slot / per;
  return checked_piece(c, r, b, slot - b * per, b * r.even, (b + 1) * r.even, c.ends[b]);
}
__device__ __forceinline__ int slot_base(const BlockRows& r, int cu, int b, int shift, int extra) {
  return (min(max(cu, 0), r.rows) * r.mul >> shift) + extra * b;
}

// Called by whole warps; every lane gets the answer.  Everything that may be the answer is read before it is known which is.
// Whoever looks for the last slot reads all of cu, so offsets that do not fit are reported wherever they stand: where they descend,
// a sequence may have no slots that lead to it.
__device__ __forceinline__ BlockPiece find_piece(const sphkv_blocks& c, const BlockRows& r, int slot, int shift, int extra) {
  if (r.cu == nullptr) return even_piece(c, r, slot, shift, extra);
  int b = -1, base = 0, lo = 0, hi = 0, end = 0;
  for (int b0 = 0; b0 < c.B; b0 += 32) {
    const int i = min(b0 + (int)(threadIdx.x & 31), c.B - 1);
    const bool there = b0 + (int)(threadIdx.x & 31) < c.B;
    const int from = r.cu[i], to = r.cu[i + 1], e = c.ends[i];
    if (there && bad_rows(r, from, to)) bad_status(c, SPHKV_ST_BAD_LENGTH);
    const int mine = there ? slot_base(r, from, i, shift, extra) : 0x7fffffff;
    const unsigned below = __ballot_sync(0xffffffffu, mine <= slot);
    if (below == 0) break;
    const int last = 31 - __clz(below);
    b = b0 + last;
    base = __shfl_sync(0xffffffffu, mine, last);
    lo = __shfl_sync(0xffffffffu, from, last);
    hi = __shfl_sync(0xffffffffu, to, last);
    end = __shfl_sync(0xffffffffu, e, last);
    if (last < 31) break;
  }
  return checked_piece(c, r, b, slot - base, lo, hi, end);
}
// The same by one thread.  There is a slot for every sequence, and whoever looks for it reports that sequence's offsets.
__device__ __forceinline__ BlockPiece find_piece_alone(const sphkv_blocks& c, const BlockRows& r, int slot, int shift, int extra) {
  if (r.cu == nullptr) return even_piece(c, r, slot, shift, extra);
  if (slot < c.B && bad_rows(r, r.cu[slot], r.cu[slot + 1])) bad_status(c, SPHKV_ST_BAD_LENGTH);
  int lo = 0;  // the last sequence whose slots begin at or before this one
  if (c.B <= 32) {  // loads that do not wait for one another
#pragma unroll 8
    for (int i = 1; i < c.B; ++i) lo = slot_base(r, r.cu[i], i, shift, extra) <= slot ? i : lo;
  } else {
    int hi = c.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      (slot_base(r, r.cu[mid], mid, shift, extra) <= slot ? lo : hi) = mid;
    }
  }
  const int from = r.cu[lo], to = r.cu[lo + 1], end = c.ends[lo];
  return checked_piece(c, r, lo, slot - slot_base(r, from, lo, shift, extra), from, to, end);
}

// ---- work dealt evenly: tiles of all slots and heads in one line ------------------------------------------------
// prefix[s] = tiles of the slots before s, prefix[slots] = all; items[s]: the slot's item, which has its `tiles`.  The host has
// checked that all tiles of all heads are fewer than 2^31.  By one block, of any number of slots.
template <typename Item, typename F>
__device__ __forceinline__ void plan_tiles(int slots, uint32_t* prefix, Item* items, F item) {
  __shared__ uint32_t warp_sums[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t before = 0;
  for (int s0 = 0; s0 < slots; s0 += blockDim.x) {
    const int s = s0 + tid;
    uint32_t v = 0;
    if (s < slots) {
      const Item u = item(s);
      items[s] = u;
      v = u.tiles;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    uint32_t add = before;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) {
      if (w < warp) add += warp_sums[w];
      before += warp_sums[w];
    }
    if (s < slots) prefix[s + 1] = v + add;
    __syncthreads();
  }
  if (tid == 0) prefix[0] = 0;
}
// The same for at most kDealt slots by the first warp of every block that shares in the work: its shuffles take a third of
// what a block's barriers take, and no launch goes before.
constexpr int kDealt = 128;
template <typename Item, typename F>
__device__ __forceinline__ void deal_tiles(int slots, uint32_t* prefix, Item* items, F item) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    uint32_t before = 0;
#pragma unroll 1
    for (int s0 = 0; s0 < slots; s0 += 32) {
      uint32_t v = 0;
      if (s0 + lane < slots) {
        const Item u = item(s0 + lane);
        items[s0 + lane] = u;
        v = u.tiles;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
      }
      if (s0 + lane < slots) prefix[s0 + lane + 1] = before + v;
      before += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) prefix[0] = 0;
  }
  __syncthreads();
}
// Tiles for each worker in turn, none without while there are tiles: a slot's segments are those of consecutive workers.
struct Shares {
  uint32_t n, per, more;  // workers with tiles; tiles of each; the first `more` have one more
  __device__ __forceinline__ Shares(uint32_t total, uint32_t workers) {
    n = min(workers, total);
    per = n ? total / n : 0;
    more = total - per * n;
  }
  __device__ __forceinline__ uint32_t start(uint32_t w) const { return w * per + min(w, more); }
  __device__ __forceinline__ uint32_t owner(uint32_t tile) const {
    const uint32_t large = more * (per + 1);
    return tile < large ? tile / (per + 1) : more + (tile - large) / per;
  }
};
__device__ __forceinline__ int slot_at(const uint32_t* prefix, int slots, uint32_t tile) {  // prefix[s] <= tile < prefix[s + 1]
  int lo = 0, hi = slots;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    (prefix[mid] <= tile ? lo : hi) = mid;
  }
  return lo;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ---- 8-bit codes -> f16 pairs, exactly ------------------------------------------------------------------
// whole numbers: f16 1024 + (code + 128) has the biased code as its low byte
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
// four codes of one word -> (0, 1) and (2, 3)
template <bool I8>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& p01, uint32_t& p23) {
  if (I8) {
    const uint32_t u = w ^ 0x80808080u;
    p01 = hsub2(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u);
    p23 = hsub2(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u);
  } else {
    p01 = e4m3x2_to_f16x2((uint16_t)w);
    p23 = e4m3x2_to_f16x2((uint16_t)(w >> 16));
  }
}

// one box of a 2-D tensor map, global -> this CTA's shared memory
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "l"(policy)
      : "memory");
}

// ---- host ------------------------------------------------------------------------------------------------
int check_blocks(const sphkv_blocks* c, const char* what);
int block_rows(BlockRows& r, const sphkv_blocks* c, const int32_t* cu, int64_t rows, const char* what);
// codes as a matrix [n_pages * Hkv * page_size][dh] of bytes, boxes of `box_rows` whole rows, swizzled in shared memory over
// a row's bytes
int make_codes_map(CUtensorMap* map, const sphkv_blocks& c, void* codes, int box_rows, const char* what);
int check_queries(const sphkv_blocks& c, const void* q, int q_dtype, const void* out, const float* out_partial, int out_dtype, int Hq,
                  float sm_scale, const char* what);
// attention of up to eight query rows a unit: 1 << tshift tokens of a sequence, at most 1 << tokens_shift(group)
int tokens_shift(int group);
int few_queries(const sphkv_blocks& c, const BlockRows& r, const void* q, int q_dtype, int64_t q_row_stride, int64_t q_head_stride,
                const int32_t* first, void* out, int out_dtype, float* out_partial, void* scratch, int64_t scratch_bytes, int Hq,
                float sm_scale, int tshift, const char* what, cudaStream_t st);
int64_t few_queries_scratch(int64_t rows, int B, int Hkv, int dh, int tshift, int sms);

}  // namespace sphkv
