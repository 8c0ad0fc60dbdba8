// Attention over the 8-bit block cache for few queries a sequence: one token (decode), or a handful.
//
// A unit is up to eight query rows that share a KV head (the head's group, times as many tokens as fit).  Per key and KV head
// 2 dh bytes are read and 4 dh operations done for each row, so memory bounds it; what the kernel has to watch is
// instructions, since every code has to become an f16 first.  Both products therefore run on the tensor cores with the
// cache as the 16-row operand, straight from the codes' own bytes: codes are exact in f16, and the freedom to number an
// operand's rows and depth lets a lane take whole 16-byte chunks.
//   logits[16 keys x 8 rows] = codes[16 x dh] . q        (lane 4g + j: keys g, g + 8; dims dh/4 j ..)
//   out[dh x 8 rows] += codes^T[dh x 16] . weights       (lane 4g + j: dims dh/8 g ..; keys 2j, 2j + 1, 2j + 8, 2j + 9)
// The logits' layout (row 2j, 2j + 1 of keys g, g + 8) becomes the weights' operand by four transposes of 8 x 8.
// Precision: a query row is scaled by a power of two so that its largest element lies in [2^13, 2^14): bf16 and f16 rows are
// exact in f16 then, fp32 rows go in as hi + lo (22 bits); weights are hi + lo as well; sums are fp32.  A page's key scale
// multiplies its logits, its value scale its weights.  A row has two references, whole powers of two: one of its logits, for the sum of
// p, and one of logit and value scale together, for the weights p v, so that f16 has the bits of what weighs most in the row, whatever
// scales stand beside it.
//
// Work: 16-token tiles of all (unit, tile) pairs in one line, cut evenly over the CTAs; a CTA's share of a unit is a segment.
// A segment's tiles go round the CTA's warps; each warp keeps maxima, sums and outputs of its own, with its own ring of
// tiles that TMA fills (three of 4 KB: 192 KB on their way per SM), so nothing is shared until the segment's end.
//
// Measured (graph replay; codes and outputs at the copy rate of 6563 GB/s in brackets): 8 x 32768 tokens x 8 heads of 128 dims 100 us
// in int8, 97 .. 100 in e4m3 (82); 1 x 131072 58 (41); 16 x 8192 59 (41: of 128 units on 148 CTAs most CTAs have two segments, and
// a segment's beginning and end take 3 us each), two tokens each 60; 1 x 2048 of 64 dims 13, latency: 3.8 us inside the kernel
// are accounted for (work dealt 1.2, addresses and first tiles 1, tiles 0.8, warps joined 0.8), its launch and end and the second
// launch are not taken apart.  DRAM 55 % at 8 x 16384 under cold caches, issue slots 56 % (464 instructions a tile in int8, 366
// in e4m3), tensor pipe 23 %: with 16 warps neither bandwidth nor issue is full, the warps' own chains are long.
#include <cmath>

#include "blocks.cuh"

namespace sphkv {

constexpr int kBdWarps = 16, kBdThreads = 32 * kBdWarps;
constexpr float kLazy = 8.f;   // a reference moves when a logit passes it by 2^8
constexpr int kWeightLog = 6;  // a weight at its reference is 2^6 and none is above 2^14: f16 keeps 22 bits (hi + lo) of those above 2^-3

struct BdArgs {
  alignas(64) CUtensorMap k_map, v_map;
  sphkv_blocks c;
  BlockRows r;
  const void* q;
  int64_t q_row_stride, q_head_stride;
  const int32_t* first;
  void* out;
  float* out_partial;
  const uint32_t* prefix;  // tiles of the slots before each, where a launch has summed them; else NULL
  const struct BdUnit* items;
  int4* spans;            // of each unit: first worker, workers, its queries' first row, tokens
  float* parts;           // [workers + units][8][dh + 2]
  int q_dtype, out_dtype, Hq, group, slots, tshift, workers;
  float scale_log2;       // sm_scale * log2 e
};

template <int DH>
struct Bd {
  static constexpr int kTile = 16 * DH;                            // bytes of a tile's keys, or values
  static constexpr int kStages = DH == 128 ? 3 : 6;
  static constexpr int kRing = 2 * kTile * kStages;                // of a warp
  static constexpr int kGroupDims = DH / 8;                        // output dims of a lane
  static constexpr int kCol = 8 * (kGroupDims + 2) + 4;            // floats of an output row in shared memory: no bank twice
  static constexpr int kPrefixOff = kBdWarps * kRing;
  static constexpr int kItemsOff = kPrefixOff + (kDealt + 4) * 4;
  static constexpr int kStatOff = kItemsOff + kDealt * 32;
  static constexpr int kStat = 5 * 8;                              // floats of a warp: references, sums, true maxima, the weights' references, factors
  static constexpr int kQOff = kStatOff + (kBdWarps * kStat + 8 * 4) * 4;
  static constexpr int kQRow = 2 * (DH + 8);                       // bytes of a row of queries in f16
  static constexpr int kQ = 2 * 8 * kQRow + 32;                    // hi, lo, factors
  static constexpr int kBarOff = kQOff + kQ;
  static constexpr int kSmem = kBarOff + kBdWarps * kStages * 8 + 1024;
};
static_assert(Bd<128>::kSmem <= 232448 && Bd<64>::kSmem <= 232448, "shared memory of a CTA");
static_assert(8 * Bd<128>::kCol * 4 <= Bd<128>::kRing, "a warp's outputs are joined in its ring's place");

// The keys of one unit's queries.
struct BdUnit {
  int b, row0, tokens;      // dense rows of the unit's queries; tokens = 0: none
  int pos0, first, limit;   // position of the first of them; keys first .. limit - 1 are seen by some
  int tile0, tiles;
};
__device__ __forceinline__ BdUnit unit_of(const BdArgs& a, const BlockPiece& p) {
  BdUnit u = {p.b, 0, 0, 0, 0, 0, 0, 0};
  const int i0 = p.j << a.tshift;
  if (p.b < 0 || i0 >= p.n) return u;
  u.row0 = p.row0 + i0;
  u.tokens = min(1 << a.tshift, p.n - i0);
  if (p.end < 0) return u;
  u.pos0 = p.end - p.n + i0;
  u.limit = u.pos0 + u.tokens;
  u.first = a.first ? min(max(a.first[p.b], 0), u.limit) : 0;
  u.tile0 = u.first >> 4;
  u.tiles = u.first < u.limit ? ((u.limit + 15) >> 4) - u.tile0 : 0;
  return u;
}

static_assert(sizeof(BdUnit) == 32, "a slot's place");
__device__ __forceinline__ BdUnit unit_of_slot(const BdArgs& a, int s) { return unit_of(a, find_piece_alone(a.c, a.r, s, a.tshift, 1)); }
__global__ void __launch_bounds__(1024) blocks_plan_kernel(const __grid_constant__ BdArgs a, uint32_t* prefix, BdUnit* items) {
  griddep_wait();
  plan_tiles(a.slots, prefix, items, [&](int s) { return unit_of_slot(a, s); });
}
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float power_of_2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// A difference of two references, which are whole, as far as it matters: a row's logits are at most 2^129 times as heavy with
// their value scales, and where they are 2^240 times as heavy without them, p of all that is not 0 is below 2^-126.
__device__ __forceinline__ int exponent(float d) { return (int)fminf(fmaxf(d, -240.f), 240.f); }
// p * vs * 2^(kWeightLog + e), which is at most 2^14 where p and vs are not 0, though vs * 2^e may be beyond fp32.  Not in line:
// a rare one.  (Scales below fp32's normal numbers are no part of the references, and count as 0.)
static __device__ __noinline__ float far_weight(float p, float vs, int e) {
  if (vs < 0x1p-126f) return p * 0.f;
  if (p == 0.f && vs < INFINITY) return 0.f;
  const int half = e / 2;
  return p * power_of_2(half) * power_of_2(kWeightLog) * vs * power_of_2(e - half);
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint4 lds_u4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 lds_u2(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
// where 16-byte chunk c of row t lies in a tile that a tensor copy has swizzled
template <int DH>
__device__ __forceinline__ uint32_t chunk_at(int t, int c) {
  return DH == 128 ? t * 128 + ((c ^ (t & 7)) << 4) : t * 64 + ((c ^ ((t >> 1) & 3)) << 4);
}
// codes of two keys at four dims -> f16 pairs (key 0, key 1) for each dim
template <bool I8>
__device__ __forceinline__ void pair_codes(uint32_t k0, uint32_t k1, uint32_t (&d)[4]) {
  const uint32_t lo = __byte_perm(k0, k1, 0x5140), hi = __byte_perm(k0, k1, 0x7362);
  codes_to_f16<I8>(lo, d[0], d[1]);
  codes_to_f16<I8>(hi, d[2], d[3]);
}

template <int DH, bool I8, bool QLO>
__global__ void __launch_bounds__(kBdThreads, 1) blocks_decode_kernel(const __grid_constant__ BdArgs a) {
  using L = Bd<DH>;
  constexpr int S = L::kStages, KS = DH / 16, GD = L::kGroupDims, W4 = GD / 4;  // words of a value row per lane
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
  constexpr int WARPS = kBdWarps;
  const uint32_t ring = smem_u32(smem) + warp * L::kRing;
  const uint32_t bars = smem_u32(smem) + L::kBarOff + warp * S * 8;
  float* const stats = reinterpret_cast<float*>(smem + L::kStatOff);
  float4* const cols_of = reinterpret_cast<float4*>(stats + WARPS * L::kStat);  // of a query row: reference, sum, true maximum, the weights' reference
  float* const joined = reinterpret_cast<float*>(smem);  // a warp's outputs: in its ring's place
  constexpr int JOIN = L::kRing / 4;
  const uint32_t q_at = smem_u32(smem) + L::kQOff;  // the segment's queries
  float* const q_factor = reinterpret_cast<float*>(smem + L::kQOff + 2 * 8 * L::kQRow);
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < S; ++s) mbar_init(bars + 8 * s, 1);
    fence_async_smem();
  }
  __syncthreads();
  griddep_wait();
  const uint32_t* prefix = a.prefix;
  const BdUnit* items = a.items;
  if (prefix == nullptr) {
    uint32_t* const at = reinterpret_cast<uint32_t*>(smem + L::kPrefixOff);
    BdUnit* const of = reinterpret_cast<BdUnit*>(smem + L::kItemsOff);
    deal_tiles(a.slots, at, of, [&](int s) { return unit_of_slot(a, s); });
    prefix = at;
    items = of;
  }
  const Shares shares(prefix[a.slots] * a.c.Hkv, a.workers);
  for (int s = blockIdx.x; s < a.slots; s += gridDim.x)  // units without keys: zeros, by the second launch
    if (items[s].tiles == 0 && tid < a.c.Hkv)
      for (int h = tid; h < a.c.Hkv; h += kBdThreads) a.spans[s * a.c.Hkv + h] = make_int4(0, 0, items[s].row0, items[s].tokens);
  const uint32_t worker = blockIdx.x;
  uint32_t pos = worker < shares.n ? shares.start(worker) : 0;
  const uint32_t stop = worker < shares.n ? shares.start(worker + 1) : 0;
  const uint64_t policy = policy_evict_first();
  const int shift = 31 - __clz(a.c.page_size);
  uint32_t issued = 0, taken = 0;  // tiles since the kernel began: stage = n % S, the barrier's phase n / S
  bool lost = false;

  while (pos < stop) {
    // ---- the segment ----
    const int slot = slot_at(prefix, a.slots, pos / a.c.Hkv);
    const BdUnit u = items[slot];
    const uint32_t in_slot = pos - prefix[slot] * a.c.Hkv;
    const int head = in_slot / (uint32_t)u.tiles, from = in_slot - head * u.tiles;
    const int count = min((uint32_t)(u.tiles - from), stop - pos);
    const int unit = slot * a.c.Hkv + head;
    if (from == 0 && tid == 0)
      a.spans[unit] = make_int4(worker, shares.owner(pos + u.tiles - 1) - worker + 1, u.row0, u.tokens);
    pos += count;
    const int cols = u.tokens * a.group;

    // ---- queries, a warp to a row: asked for here, used behind the tiles' addresses ----
    constexpr int QD = DH / 32;  // dims of a lane
    float qv[QD];
    const bool q_row = warp < cols;
    if (q_row) {
      const int tok = warp / a.group, h = head * a.group + warp - tok * a.group;
      const int64_t at = (int64_t)(u.row0 + tok) * a.q_row_stride + (int64_t)h * a.q_head_stride + QD * lane;
#pragma unroll
      for (int i = 0; i < QD; ++i) qv[i] = load_as_float(a.q, a.q_dtype, at + i);
    }
    // ---- where this warp's tiles lie: lane i holds tile 32 r + i of them ----
    const int mine = warp < count ? (count - warp + WARPS - 1) / WARPS : 0;
    const int32_t* table = a.c.block_table + (int64_t)u.b * a.c.max_blocks;
    struct Meta {
      int row;  // of the pools; negative: a bad table entry
      float ks, vs;
    };
    auto lookup = [&](int k) {
      Meta m = {0, 0.f, 0.f};
      if (k >= mine) return m;
      const int tok = (u.tile0 + from + warp + k * WARPS) << 4;
      const int page = table[tok >> shift];
      if (page < 0 || page >= a.c.n_pages) {
        bad_status(a.c, SPHKV_ST_BAD_BLOCK);
        m.row = -1;
        return m;
      }
      const int at = page * a.c.Hkv + head;
      m.row = (at << shift) + (tok & (a.c.page_size - 1));
      m.ks = a.c.k_scale[at];
      m.vs = a.c.v_scale[at];
      return m;
    };
    Meta cur = lookup(lane), nxt = lookup(32 + lane);
    auto issue = [&](int k, int base) {  // tile k; `cur` holds tiles base .. base + 31
      const int row = __shfl_sync(0xffffffffu, k - base < 32 ? cur.row : nxt.row, k & 31);
      if (lane == 0) {
        const uint32_t s = issued % S, bar = bars + 8 * s, at = ring + s * 2 * L::kTile;
        mbar_expect_tx(bar, 2 * L::kTile);
        tma_load_2d(at, &a.k_map, 0, max(row, 0), bar, policy);
        tma_load_2d(at + L::kTile, &a.v_map, 0, max(row, 0), bar, policy);
      }
      ++issued;
    };
    if (!lost)
      for (int k = 0; k < min(S, mine); ++k) issue(k, 0);

    // ---- the rows in f16, scaled by powers of two; then lane 4g + j takes dims DH/4 j .. of row g ----
    if (warp < 8) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < QD; ++i) {
        if (!q_row) qv[i] = 0.f;
        top = isnan(qv[i]) ? INFINITY : fmaxf(top, fabsf(qv[i]));
      }
      const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
      int e = (int)(bits >> 23);
      e = e == 255 ? 140 : max(e, 14);  // infinities and NaN go in as they are
      const float up = __uint_as_float((uint32_t)(267 - e) << 23);
      if (lane == 0) q_factor[warp] = __uint_as_float((uint32_t)(e - 13) << 23) * a.scale_log2;
#pragma unroll
      for (int i = 0; i < QD; i += 2) {
        uint32_t hi, lo;
        split_f16x2(qv[i] * up, qv[i + 1] * up, hi, lo);
        const uint32_t to = q_at + warp * L::kQRow + 2 * (QD * lane + i);
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(to), "r"(hi) : "memory");
        if constexpr (QLO) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + 8 * L::kQRow), "r"(lo) : "memory");
      }
    }
    __syncthreads();
    uint32_t qh[KS][2], ql[QLO ? KS : 1][2];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint32_t from = q_at + g * L::kQRow + 2 * ((DH / 4) * j + 4 * s);
      const uint2 h = lds_u2(from);
      qh[s][0] = h.x, qh[s][1] = h.y;
      if constexpr (QLO) {
        const uint2 l = lds_u2(from + 8 * L::kQRow);
        ql[s][0] = l.x, ql[s][1] = l.y;
      }
    }
    const float f0 = q_factor[2 * j], f1 = q_factor[2 * j + 1];  // logit factors of rows 2j, 2j + 1; where their keys end
    const int lim0 = 2 * j < cols ? u.pos0 + 2 * j / a.group + 1 : u.limit;
    const int lim1 = 2 * j + 1 < cols ? u.pos0 + (2 * j + 1) / a.group + 1 : u.limit;
    const int least = u.tokens > 1 ? u.pos0 + 1 : u.limit;

    float acc[KS][4];  // [DH / 16 row tiles of dims]
#pragma unroll
    for (int i = 0; i < KS; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const float kNone = -3.402823466e38f;
    float m0 = kNone, m1 = kNone, l0 = 0.f, l1 = 0.f, t0 = -INFINITY, t1 = -INFINITY;
    float v0 = kNone, v1 = kNone;  // the weights' references
    float up0 = 1.f, up1 = 1.f;    // 2^kWeightLog * 2^(m - v), where
    bool far = false;              // no row has its references more than 2^60 apart

    for (int k = 0, base = 0; k < mine; ++k) {
      if (k - base == 32) {
        base += 32;
        cur = nxt;
        nxt = lookup(base + 32 + lane);
      }
      const int src = k & 31;
      const int row = __shfl_sync(0xffffffffu, cur.row, src);
      const float ks = __shfl_sync(0xffffffffu, cur.ks, src), vs = __shfl_sync(0xffffffffu, cur.vs, src);
      const uint32_t stage = taken % S;
      if (!lost && !mbar_wait(bars + 8 * stage, (taken / S) & 1)) {
        lost = true;
        bad_status(a.c, SPHKV_ST_TIMEOUT);
      }
      if (lost) break;
      ++taken;
      const uint32_t kt = ring + stage * 2 * L::kTile, vt = kt + L::kTile;

      // logits
      float c[2][4] = {};
#pragma unroll
      for (int q4 = 0; q4 < DH / 64; ++q4) {
        const uint4 x = lds_u4(kt + chunk_at<DH>(g, (DH / 64) * j + q4)), y = lds_u4(kt + chunk_at<DH>(g + 8, (DH / 64) * j + q4));
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int s = 4 * q4 + w;
          uint32_t a0, a1, a2, a3;
          codes_to_f16<I8>(xw[w], a0, a2);
          codes_to_f16<I8>(yw[w], a1, a3);
          mma_16x8x16(c[w & 1], a0, a1, a2, a3, qh[s][0], qh[s][1]);
          if constexpr (QLO) mma_16x8x16(c[w & 1], a0, a1, a2, a3, ql[s][0], ql[s][1]);
        }
      }
      uint32_t vw[4][W4];  // keys 2j, 2j + 1, 2j + 8, 2j + 9; dims GD g ..
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int t = 2 * j + (n & 1) + 8 * (n >> 1);
        if constexpr (DH == 128) {
          const uint4 v = lds_u4(vt + chunk_at<DH>(t, g));
          vw[n][0] = v.x, vw[n][1] = v.y, vw[n][2] = v.z, vw[n][3] = v.w;
        } else {
          const uint2 v = lds_u2(vt + chunk_at<DH>(t, g >> 1) + 8 * (g & 1));
          vw[n][0] = v.x, vw[n][1] = v.y;
        }
      }
      __syncwarp();
      if (k + S < mine) issue(k + S, base);

      const float e0 = f0 * ks, e1 = f1 * ks;
      float x[4] = {(c[0][0] + c[1][0]) * e0, (c[0][1] + c[1][1]) * e1, (c[0][2] + c[1][2]) * e0, (c[0][3] + c[1][3]) * e1};
      const int tok = (u.tile0 + from + warp + k * WARPS) << 4;
      const bool edge = row < 0 || tok < u.first || tok + 16 > least;
      bool seen[4] = {true, true, true, true};
      if (edge) {  // some keys of the tile are not seen by every row, or by none
        const int ta = tok + g, tb = ta + 8;
        seen[0] = row >= 0 && ta >= u.first && ta < lim0;
        seen[1] = row >= 0 && ta >= u.first && ta < lim1;
        seen[2] = row >= 0 && tb >= u.first && tb < lim0;
        seen[3] = row >= 0 && tb >= u.first && tb < lim1;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!seen[i]) x[i] = -INFINITY;
#pragma unroll
        for (int n = 0; n < 4; ++n) {  // what lies behind the last token may be any byte
          const int t = tok + 2 * j + (n & 1) + 8 * (n >> 1);
          if (row < 0 || t < u.first || t >= u.limit)
#pragma unroll
            for (int w = 0; w < W4; ++w) vw[n][w] = 0;
        }
      }
      const float x0 = fmaxf(x[0], x[2]), x1 = fmaxf(x[1], x[3]);
      t0 = fmaxf(t0, x0);
      t1 = fmaxf(t1, x1);
      const float lv = lg2(vs);  // approximate: between 2^14 and the largest f16 is room
      if (__any_sync(0xffffffffu, x0 > fminf(m0, v0 - lv) + kLazy || x1 > fminf(m1, v1 - lv) + kLazy)) {
        float n0 = x0, n1 = x1;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
          n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
        }
        far = false;
        auto move = [&](float n, float& m, float& l, float& v, float& up) {  // what the weights so far are multiplied by
          const float to = fmaxf(ceilf(n), m), v_to = fmaxf(ceilf(n + lv), v), r = ex2(v - v_to);
          const int e = exponent(to - v_to);
          l *= ex2(m - to);
          m = to;
          v = v_to;
          up = power_of_2(min(max(e, -60), 60) + kWeightLog);
          far |= abs(e) > 60;
          return r;
        };
        const float r0 = move(n0, m0, l0, v0, up0), r1 = move(n1, m1, l1, v1, up1);
#pragma unroll
        for (int i = 0; i < KS; ++i) acc[i][0] *= r0, acc[i][1] *= r1, acc[i][2] *= r0, acc[i][3] *= r1;
      }
      float w[4] = {ex2(x[0] - m0), ex2(x[1] - m1), ex2(x[2] - m0), ex2(x[3] - m1)};
      l0 += w[0] + w[2];
      l1 += w[1] + w[3];
      if (far || vs > 0x1p60f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = far_weight(w[i], vs, exponent(i & 1 ? m1 - v1 : m0 - v0));
      } else {
        const float ve0 = vs * up0, ve1 = vs * up1;
        w[0] *= ve0, w[1] *= ve1, w[2] *= ve0, w[3] *= ve1;
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!seen[i]) w[i] = 0.f;  // the scale may be NaN
      }
      uint32_t ph[2], pl[2];
      split_f16x2(w[0], w[1], ph[0], pl[0]);
      split_f16x2(w[2], w[3], ph[1], pl[1]);
      const uint32_t bh0 = transposed(ph[0]), bh1 = transposed(ph[1]), bl0 = transposed(pl[0]), bl1 = transposed(pl[1]);
#pragma unroll
      for (int q4 = 0; q4 < W4; ++q4) {  // four dims of the lane: two row tiles
        uint32_t d01[4], d89[4];
        pair_codes<I8>(vw[0][q4], vw[1][q4], d01);
        pair_codes<I8>(vw[2][q4], vw[3][q4], d89);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mma_16x8x16(acc[2 * q4 + h], d01[2 * h], d01[2 * h + 1], d89[2 * h], d89[2 * h + 1], bh0, bh1);
          mma_16x8x16(acc[2 * q4 + h], d01[2 * h], d01[2 * h + 1], d89[2 * h], d89[2 * h + 1], bl0, bl1);
        }
      }
    }

    // ---- the warps are joined ----
    {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, o);
        l1 += __shfl_xor_sync(0xffffffffu, l1, o);
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
      }
      float* const st = stats + warp * L::kStat;
      if (g == 0) {
        st[2 * j] = m0, st[2 * j + 1] = m1;
        st[8 + 2 * j] = l0, st[9 + 2 * j] = l1;
        st[16 + 2 * j] = t0, st[17 + 2 * j] = t1;
        st[24 + 2 * j] = v0, st[25 + 2 * j] = v1;
      }
      float* const mine_at = joined + warp * JOIN + g * (GD + 2);  // this warp has taken every tile of its own
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        *reinterpret_cast<float2*>(mine_at + 2 * j * L::kCol + 2 * i) = make_float2(acc[i][0], acc[i][2]);
        *reinterpret_cast<float2*>(mine_at + (2 * j + 1) * L::kCol + 2 * i) = make_float2(acc[i][1], acc[i][3]);
      }
      __syncthreads();
      const int n_warps = min(count, WARPS);
      for (int col = warp; col < cols; col += WARPS) {  // a warp to a query row: lane w looks after warp w
        const float* const of = stats + (lane % WARPS) * L::kStat + col;
        const bool have = lane < n_warps;
        float top = have ? of[0] : kNone, true_top = have ? of[16] : -INFINITY, v_top = have ? of[24] : kNone;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          true_top = fmaxf(true_top, __shfl_xor_sync(0xffffffffu, true_top, o));
          v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, o));
        }
        const float f = have ? ex2(of[0] - top) : 0.f;
        float sum = have ? of[8] * f : 0.f;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (have) stats[lane * L::kStat + 32 + col] = ex2(of[24] - v_top);
        if (lane == 0) cols_of[col] = make_float4(top, sum, true_top, v_top);
      }
      __syncthreads();
      const bool whole = count == u.tiles;
      float* const part = a.parts + (int64_t)(worker + unit) * 8 * (DH + 2);
      for (int i = tid; i < cols * DH; i += kBdThreads) {
        const int col = i / DH, d = i - col * DH;
        const float* const from = joined + col * L::kCol + (d / GD) * (GD + 2) + d % GD;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
          if (w < n_warps) v += from[w * JOIN] * stats[w * L::kStat + 32 + col];
        const float4 of = cols_of[col];
        const float top = of.x, sum = of.y, true_top = of.z;
        const float to_true = true_top == -INFINITY ? 0.f : ex2(top - true_top);
        const int e = exponent(of.w - top) - kWeightLog;
        v = v * power_of_2(e >> 1) * power_of_2(e - (e >> 1));
        if (whole) {
          const int tok = col / a.group, h = head * a.group + col - tok * a.group;
          const int64_t at = (int64_t)(u.row0 + tok) * a.Hq + h;
          if (a.out) store_from_float(a.out, a.out_dtype, at * DH + d, sum == 0.f ? 0.f : v / sum);
          if (a.out_partial) {
            float* o = a.out_partial + at * (DH + 2);
            o[2 + d] = v * to_true;
            if (d == 0) o[0] = true_top * kLn2, o[1] = sum * to_true;
          }
        } else {
          part[col * (DH + 2) + 2 + d] = v * to_true;
          if (d == 0) part[col * (DH + 2)] = true_top, part[col * (DH + 2) + 1] = sum * to_true;
        }
      }
      __syncthreads();
      fence_async_smem();  // the next segment's copies come in through the other proxy
      __syncthreads();
    }
  }
  if (lost) {  // copies that are still on their way
    for (; taken != issued; ++taken) (void)mbar_wait(bars + 8 * (taken % S), (taken / S) & 1);
  }
}

// A block per query row, a thread per dim: joins the segments of units that more than one worker had, and writes the rows of
// units without keys.
constexpr int kBdParts = 128;  // segments whose factors are in shared memory at a time
template <int DH>
__global__ void __launch_bounds__(DH) blocks_merge_kernel(const __grid_constant__ BdArgs a) {
  __shared__ float factor[kBdParts], tops[DH / 32], adds[DH / 32];
  griddep_launch();
  const int unit = blockIdx.x, col = blockIdx.y;
  const int4 span = a.spans[unit];
  const int first = span.x, n = span.y, row0 = span.z;
  if (n == 1 || col >= span.w * a.group) return;  // one worker: it has written its unit
  const int head = unit % a.c.Hkv;
  const int d = threadIdx.x, warp = d >> 5, lane = d & 31;
  constexpr int STEP = 8 * (DH + 2);
  const float* const rows = a.parts + (int64_t)(first + unit) * STEP + col * (DH + 2);
  float top = -INFINITY;
  for (int p = d; p < n; p += DH) top = fmaxf(top, rows[p * STEP]);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < DH / 32; ++w) top = fmaxf(top, tops[w]);
  float sum = 0.f, v = 0.f;
  for (int p0 = 0; p0 < n; p0 += kBdParts) {
    const int here = min(kBdParts, n - p0);
    if (p0 > 0) __syncthreads();
    for (int p = d; p < here; p += DH) {
      const float* const row = rows + (p0 + p) * STEP;
      const float f = row[0] == -INFINITY ? 0.f : ex2(row[0] - top);
      factor[p] = f;
      sum += row[1] * f;
    }
    __syncthreads();
    const float* const from = rows + p0 * STEP + 2 + d;
#pragma unroll 8
    for (int p = 0; p < here; ++p) v += from[p * STEP] * factor[p];
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) adds[warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < DH / 32; ++w) sum += adds[w];
  const int tok = col / a.group, h = head * a.group + col - tok * a.group;
  const int64_t at = (int64_t)(row0 + tok) * a.Hq + h;
  if (a.out) store_from_float(a.out, a.out_dtype, at * DH + d, sum == 0.f ? 0.f : v / sum);
  if (a.out_partial) {
    float* const o = a.out_partial + at * (DH + 2);
    o[2 + d] = v;
    if (d == 0) o[0] = top == -INFINITY ? -INFINITY : top * kLn2, o[1] = sum;
  }
}

int tokens_shift(int group) { return group == 1 ? 3 : group == 2 ? 2 : group <= 4 ? 1 : 0; }
static int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

static int64_t bd_scratch(int64_t slots, int Hkv, int dh, int workers) {
  return align256((slots + 1) * 4) + align256(slots * (int64_t)sizeof(BdUnit)) + align256(slots * Hkv * 16) + (workers + slots * Hkv) * 8 * (dh + 2) * 4;
}

template <int DH, bool I8, bool QLO>
static int launch_bd(const BdArgs& a, int ctas, cudaStream_t st) {
  static SmemOptIn opt_in;
  auto kern = blocks_decode_kernel<DH, I8, QLO>;
  if (int rc = ensure_dynamic_smem(opt_in, (const void*)kern, Bd<DH>::kSmem, "blocks_decode")) return rc;
  (void)launch_overlapped(kern, dim3(ctas), dim3(kBdThreads), Bd<DH>::kSmem, st, a);
  return check_launch("blocks_decode_kernel");
}
template <int DH>
static int launch_bd_types(const BdArgs& a, int ctas, cudaStream_t st) {
  const bool i8 = a.c.store == SPHKV_BLOCKS_I8;
  if (a.q_dtype == SPHKV_F32) return i8 ? launch_bd<DH, true, true>(a, ctas, st) : launch_bd<DH, false, true>(a, ctas, st);
  return i8 ? launch_bd<DH, true, false>(a, ctas, st) : launch_bd<DH, false, false>(a, ctas, st);
}

// a has the cache, rows, queries and outputs
static int run_bd(BdArgs& a, void* scratch, int64_t scratch_bytes, const char* what, cudaStream_t st) {
  const int sms = sm_count_current_device();
  if (sms <= 0) return sms;
  const int64_t slots = block_slots(a.r, a.c.B, a.tshift, 1);
  if (slots == 0) return 0;
  // tiles of all units are counted in 32 bits
  SPHKV_REQUIRE((double)slots * a.c.Hkv * ((int64_t)a.c.max_blocks * (a.c.page_size / 16) + 1) < 2147483648.0, SPHKV_E_LIMIT,
                "%s: too many (sequence, head, token)s for one launch", what);
  a.slots = (int)slots;
  a.workers = sms;
  const int64_t need = bd_scratch(slots, a.c.Hkv, a.c.dh, a.workers);
  SPHKV_REQUIRE(scratch != nullptr && scratch_bytes >= need, SPHKV_E_SCRATCH, "%s: scratch %lld B < %lld B", what,
                (long long)scratch_bytes, (long long)need);
  SPHKV_REQUIRE(((uintptr_t)scratch & 255) == 0, SPHKV_E_ALIGN, "%s: scratch needs 256 B", what);
  uint8_t* const items_at = reinterpret_cast<uint8_t*>(scratch) + align256((slots + 1) * 4);
  a.spans = reinterpret_cast<int4*>(items_at + align256(slots * (int64_t)sizeof(BdUnit)));
  a.parts = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.spans) + align256(slots * a.c.Hkv * 16));
  a.prefix = nullptr;
  a.items = nullptr;
  if (int rc = make_codes_map(&a.k_map, a.c, a.c.k_codes, 16, what)) return rc;
  if (int rc = make_codes_map(&a.v_map, a.c, a.c.v_codes, 16, what)) return rc;
  if (slots > kDealt) {
    uint32_t* const prefix = reinterpret_cast<uint32_t*>(scratch);
    BdUnit* const items = reinterpret_cast<BdUnit*>(items_at);
    (void)launch_overlapped(blocks_plan_kernel, dim3(1), dim3(1024), 0, st, a, prefix, items);
    if (int rc = check_launch("blocks_plan_kernel")) return rc;
    a.prefix = prefix;
    a.items = items;
  }
  if (int rc = a.c.dh == 128 ? launch_bd_types<128>(a, sms, st) : launch_bd_types<64>(a, sms, st)) return rc;
  const dim3 grid((unsigned)(slots * a.c.Hkv), (unsigned)(a.group << a.tshift));
  // a plain launch: one that may come in early is 2.5 us slower (its blocks wait where the next call's would begin)
  if (a.c.dh == 128)
    blocks_merge_kernel<128><<<grid, 128, 0, st>>>(a);
  else
    blocks_merge_kernel<64><<<grid, 64, 0, st>>>(a);
  return check_launch("blocks_merge_kernel");
}

int check_queries(const sphkv_blocks& c, const void* q, int q_dtype, const void* out, const float* out_partial, int out_dtype, int Hq,
                  float sm_scale, const char* what) {
  SPHKV_REQUIRE(std::isfinite(sm_scale), SPHKV_E_ARG, "%s: sm_scale=%g", what, (double)sm_scale);
  SPHKV_REQUIRE(out || out_partial, SPHKV_E_ARG, "%s: no output", what);
  SPHKV_REQUIRE(q_dtype >= 0 && q_dtype <= 2 && out_dtype >= 0 && out_dtype <= 2, SPHKV_E_DTYPE, "%s: q_dtype=%d out_dtype=%d", what,
                q_dtype, out_dtype);
  SPHKV_REQUIRE(Hq > 0 && Hq % c.Hkv == 0, SPHKV_E_ARG, "%s: Hq=%d Hkv=%d", what, Hq, c.Hkv);
  SPHKV_REQUIRE(Hq / c.Hkv <= SPHKV_MAX_GQA, SPHKV_E_LIMIT, "%s: %d query heads per KV head (max %d)", what, Hq / c.Hkv, SPHKV_MAX_GQA);
  const int64_t q_size = q_dtype == SPHKV_F32 ? 4 : 2, o_size = out_dtype == SPHKV_F32 ? 4 : 2;
  SPHKV_REQUIRE(((uintptr_t)q & (q_size - 1)) == 0 && ((uintptr_t)out & (o_size - 1)) == 0 && ((uintptr_t)out_partial & 3) == 0,
                SPHKV_E_ALIGN, "%s: q or an output is not on an element's boundary", what);
  return 0;
}

// Attention of the queries of `r` through this kernel.
int few_queries(const sphkv_blocks& c, const BlockRows& r, const void* q, int q_dtype, int64_t q_row_stride, int64_t q_head_stride,
                const int32_t* first, void* out, int out_dtype, float* out_partial, void* scratch, int64_t scratch_bytes, int Hq,
                float sm_scale, int tshift, const char* what, cudaStream_t st) {
  BdArgs a = {};
  a.c = c;
  a.r = r;
  a.q = q;
  a.q_dtype = q_dtype;
  a.q_row_stride = q_row_stride;
  a.q_head_stride = q_head_stride;
  a.first = first;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_partial = out_partial;
  a.Hq = Hq;
  a.group = Hq / c.Hkv;
  a.tshift = tshift;
  a.scale_log2 = sm_scale * kLog2e;
  return run_bd(a, scratch, scratch_bytes, what, st);
}
int64_t few_queries_scratch(int64_t rows, int B, int Hkv, int dh, int tshift, int sms) {
  return bd_scratch((rows >> tshift) + B, Hkv, dh, sms);
}

}  // namespace sphkv

using namespace sphkv;

extern "C" int64_t sphkv_blocks_decode_scratch_bytes(int32_t B, int32_t Hq, int32_t Hkv, int32_t dh) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > SPHKV_MAX_GQA || (dh != 64 && dh != 128)) return SPHKV_E_ARG;
  const int sms = sm_count_current_device();
  return sms <= 0 ? sms : bd_scratch(B, Hkv, dh, sms);
}

extern "C" int sphkv_blocks_decode(const sphkv_blocks* c, const void* q, int32_t q_dtype, int64_t q_row_stride, int64_t q_head_stride,
                                   const int32_t* first, void* out, int32_t out_dtype, float* out_partial, void* scratch,
                                   int64_t scratch_bytes, int32_t Hq, float sm_scale, void* stream) {
  if (int rc = check_blocks(c, "blocks_decode")) return rc;
  SPHKV_REQUIRE(q != nullptr, SPHKV_E_ARG, "blocks_decode: q is NULL");
  if (int rc = check_queries(*c, q, q_dtype, out, out_partial, out_dtype, Hq, sm_scale, "blocks_decode")) return rc;
  // one row a sequence, whatever ends[] says: one without tokens has a query all the same
  const BlockRows r = {nullptr, c->B, 1, 1, true};
  return few_queries(*c, r, q, q_dtype, q_row_stride, q_head_stride, first, out, out_dtype, out_partial, scratch, scratch_bytes, Hq,
                     sm_scale, 0, "blocks_decode", reinterpret_cast<cudaStream_t>(stream));
}
