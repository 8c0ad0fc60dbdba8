// Causal attention of many queries a sequence over the 8-bit block cache (a prompt's chunk, drafted tokens).
//
// The query rows of one KV head (tokens x group heads, flat) are cut into blocks of 256, two tensor-core tiles of 128; the
// keys into tiles of 128.  A CTA walks a block's key tiles with five kinds of warps:
//   4 + 4 warps  fetch a tile's key or value codes into registers, a tile ahead, and turn them into f16 operands in shared memory
//            (codes are exact in f16; scales stay apart), double buffered;
//   1 warp   fetches the tile's scales;
//   1 warp   issues the products: logits S_t = Q_t K^T and outputs O_t += P_t V (tcgen05, P from tensor memory), for the two
//            row tiles t in turn, so that the tensor cores work on one while the other's softmax runs;
//   8 warps  softmax, a thread to a query row, 32 keys at a time: S from tensor memory, a page's key scale times the row's
//            factor as one multiplier for its 16 keys and up, weights p v / S_v in f16 back over S as the next product's
//            operand.  The page's value scale is part of the exponent, so it costs nothing per element; the sum of p takes
//            it out again once for 16 keys.  The row's reference is of logit and value scale together, so that f16 has the bits
//            of what weighs most in the row, whatever scales it does not see; it puts the largest at 2^6 at most, is a whole
//            number, and moves only when one passes 2^14.  O and the tile's weights so far are then rescaled in place (every earlier product is complete:
//            S_t(k) is issued behind P_t V(k - 1)).
// Q rows are scaled by a power of two as in the decode kernel: bf16 and f16 queries are exact in f16.  Weights have f16's 11
// bits, rounded once, sums are fp32.  An eighth of the exponentials goes through a polynomial on the fma pipe.
//
// Work: (block, head, key tile) in one line, cut evenly over the CTAs; a block that two or more CTAs share is joined by a
// second launch.
//
// Measured: 2048 queries x 32 heads on 32768 tokens 1.10 ms in a graph, 0.97 PFLOP/s, 59 % of what cuBLAS reaches in a burst (1.26 ms,
// 52 %, through the public call in turn with other work, at the clocks that this leaves); on 8192 tokens 294 us, on their own 2048
// 223 us; five pieces of 301 .. 61 queries on up to 6001 tokens 102 us; 16 x 8192 with 4 or 8 tokens a sequence 152 us.  A pair of tiles (256 x 128) takes 5000 cycles.  The floor is 2048 for
// the products (their operands ask for 96 of shared memory's 128 bytes a cycle, the conversion for another 32) and 2048 for the
// exponentials; what is missing is in the chain of each row tile: softmax 2950 cycles (a warp alone needs 1100 for the tile, but
// there are five on each scheduler), weights seen by the products' warp 400, P V 460, S 570, logits seen 340 (1.29 ms while the next
// logits came in behind all of a step's weights).  Logits of 64 keys at a time ahead of P V, in the columns that the weights leave
// free: 1.40 ms, since a product of 64 columns takes as long as one of 128.
// Tensor pipe 38 %, issue slots 49 % (8192 tokens, cold caches), no local memory.  Local memory is what the arrangement of the roles avoids: with all of L1
// taken by shared memory a spilled word comes from L2 (1.96 ms with 512 threads and the tile's 128 logits in registers).
#include "blocks.cuh"

namespace sphkv {

constexpr int kAtRows = 256, kAtKeys = 128;
constexpr int kAtThreads = 640;  // warps 0-3, 4-7: softmax of tile 0, 1; 8-11, 12-15: keys, values to operands; 16: products;
// 17: scales; 18: what is left over; 19 has no work
constexpr int kAtProducts = 16;
// Registers of a thread: at launch; after the softmax has taken what the others gave up.  The file is four quarters, with
// five warps each (two of softmax, two of codes, one of 16 .. 19), so what goes up has to come down quarter by quarter.
constexpr int kAtRegs = 96, kAtRegsSoftmax = 136, kAtRegsCodes = 72, kAtRegsRest = 64;
static_assert(2 * kAtRegsSoftmax + 2 * kAtRegsCodes + kAtRegsRest <= 5 * kAtRegs && 20 * 32 * kAtRegs <= 65536, "registers");
// log2 of the largest weight where the reference moves, to the whole number above (below: it moves more often, 2 % more in all), and where
// it does not yet
constexpr float kAtWeight = 6.f, kAtLazy = 14.f;

struct AtArgs {
  sphkv_blocks c;
  BlockRows r;
  const void* q;
  int64_t q_row_stride, q_head_stride;
  const int32_t* first;
  void* out;
  const uint32_t* prefix;
  const struct AtItem* items;
  struct AtSpan* spans;  // [workers]: the block that a worker begins and others go on with
  float* parts;  // [workers][2][dh + 2][256]: a worker's first, cut segment and its last
  int q_dtype, out_dtype, Hq, group, slots, workers;
  bool q_vec;
  uint32_t q_sign;   // the sign of sm_scale, which the queries take: the softmax multiplies maxima, and needs a factor of 0 or more
  float scale_log2;  // its magnitude, times log2 e
};

struct AtItem {
  int b, row0;      // sequence, its first dense row
  int r0, rows;     // flat query rows of the block
  int pos0;         // position of the sequence's first query
  int first, lim[2];  // tile t sees keys first .. lim[t] - 1
  int kt0, tiles;
};
__device__ __forceinline__ AtItem item_of(const AtArgs& a, int slot) {
  const BlockPiece p = find_piece_alone(a.c, a.r, slot, 8, 1);
  AtItem u = {p.b, p.row0, 0, 0, 0, 0, {0, 0}, 0, 0};
  const int all = p.n * a.group, r0 = p.j * kAtRows;
  if (p.b < 0 || r0 >= all) return u;
  u.r0 = r0;
  u.rows = min(kAtRows, all - r0);
  if (p.end < 0) return u;
  u.pos0 = p.end - p.n;
  u.lim[0] = u.pos0 + (r0 + min(u.rows, 128) - 1) / a.group + 1;
  u.lim[1] = u.rows > 128 ? u.pos0 + (r0 + u.rows - 1) / a.group + 1 : 0;
  const int limit = max(u.lim[0], u.lim[1]);
  u.first = a.first ? min(max(a.first[p.b], 0), limit) : 0;
  u.kt0 = u.first / kAtKeys;
  u.tiles = u.first < limit ? (limit + kAtKeys - 1) / kAtKeys - u.kt0 : 0;
  return u;
}
struct AtSpan {
  int n;                      // workers; 0: no such block
  int row0, r0, rows, head;   // of AtItem
  int pad[3];
};
__global__ void __launch_bounds__(1024) blocks_attend_plan_kernel(const __grid_constant__ AtArgs a, uint32_t* prefix, AtItem* items) {
  griddep_wait();
  plan_tiles(a.slots, prefix, items, [&](int s) { return item_of(a, s); });
}

// ---- shared memory ----------------------------------------------------------------------------------------
struct AtMeta {       // of a key tile, for the softmax
  float4 of[8];       // of 16 keys: key scale; log2(value scale / S); S / value scale, which takes the value scale out of the sum of
                      // weights; unused
  float down, big;    // S before / S; S
  uint32_t bad;       // groups without a page; << 8: whose values count as zeros
  uint32_t pad;
};
constexpr int kAtWalkBytes = 112;
template <int DH>
struct At {
  static constexpr int kSlab = 128 * 128;             // 128 rows of 64 f16
  static constexpr int kOperand = kSlab * (DH / 64);  // keys or values of a tile, or a tile of queries
  static constexpr int kQ = 0, kK = 2 * kOperand, kV = kK + 2 * kOperand, kMeta = kV + 2 * kOperand;
  static constexpr int kBars = kMeta + 4 * (int)sizeof(AtMeta);
  static constexpr int kPrefix = kBars + 18 * 8;
  static constexpr int kItems = kPrefix + (kDealt + 4) * 4;
  static constexpr int kWalks = kItems + kDealt * (int)sizeof(AtItem);
  static constexpr int kSmem = kWalks + kAtThreads / 32 * kAtWalkBytes + 1024;
};
static_assert(At<128>::kSmem <= 232448, "shared memory of a CTA");
// kNext: for the n-th step of the products, keys and scales of tile n and values of tile n - 1 are there, in one barrier, since
// every wait costs the products' warp 350 cycles of its chain (1.12 ms with three); kVFull: the values alone, behind a segment's last tile.
enum { kNext = 0, kKFree = 2, kVFull = 4, kVFree = 6, kQFull = 8, kSFull = 10, kPFull = 12, kODone = 14, kLast = 16 };

__device__ __forceinline__ void tmem_ld_x32(uint32_t addr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
        "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
        "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st_x16u(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x8u(uint32_t addr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void sts_u4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 2^x without the exponential unit: x = n + r, n whole (Cody and Waite), a polynomial of degree 4 for 2^r on [-1/2, 1/2] (fitted
// by Remez' exchange: 2^-18.5 relative), and the product with 2^n, which leaves NaN as it is.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.x));  // -126
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.y));
  const float2 magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-1.f, -1.f);  // 1.5 * 2^23
  const float2 t = __fadd2_rn(x, magic);
  const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
  const float2 r = __ffma2_rn(n, minus, x);
  float2 p = make_float2(0.009570102207362652f, 0.009570102207362652f);
  p = __ffma2_rn(p, r, make_float2(0.05591785907745361f, 0.05591785907745361f));
  p = __ffma2_rn(p, r, make_float2(0.240247443318367f, 0.240247443318367f));
  p = __ffma2_rn(p, r, make_float2(0.6931217908859253f, 0.6931217908859253f));
  p = __ffma2_rn(p, r, make_float2(0.9999992847442627f, 0.9999992847442627f));
  const float2 two_n = make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                                   __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u));
  return __fmul2_rn(p, two_n);
}
// 16-byte chunk `c` (8 of dh f16) of row t: slabs of 64 columns, 128-byte swizzle
__device__ __forceinline__ uint32_t operand_at(int t, int c) { return (c >> 3) * (128 * 128) + t * 128 + (((c & 7) ^ (t & 7)) << 4); }

// The segments of one worker; every warp walks them by itself, in a place of its own in shared memory: registers are what the
// loops are short of, and local memory is L2 where shared memory takes all of L1.
struct AtWalk {
  const uint32_t* prefix;
  const AtItem* items;
  uint32_t left;  // tiles
  AtItem u;
  int slot, head, from, count, cnt[2];
  bool whole;
  __device__ __forceinline__ void begin(const AtArgs& a, uint32_t worker) {
    const Shares shares(prefix[a.slots] * a.c.Hkv, a.workers);
    left = 0;
    count = 0;
    if (worker >= shares.n) return;
    const uint32_t pos = shares.start(worker);
    left = shares.start(worker + 1) - pos;
    slot = slot_at(prefix, a.slots, pos / a.c.Hkv);
    u = items[slot];
    const uint32_t in_slot = pos - prefix[slot] * a.c.Hkv;
    head = in_slot / (uint32_t)u.tiles;
    from = in_slot - head * u.tiles;
  }
  __device__ __forceinline__ bool next(const AtArgs& a) {
    if (left == 0) return false;
    if (count > 0) {  // behind a segment: the next head, or the next block with keys
      from = 0;
      if (++head == a.c.Hkv) {
        head = 0;
        do u = items[++slot];
        while (u.tiles == 0);  // there is one: left > 0
      }
    }
    count = min((uint32_t)(u.tiles - from), left);
    left -= count;
    whole = count == u.tiles;
#pragma unroll
    for (int t = 0; t < 2; ++t) cnt[t] = min(max((u.lim[t] + kAtKeys - 1) / kAtKeys - (u.kt0 + from), 0), count);
    return true;
  }
};

static_assert(sizeof(AtWalk) <= kAtWalkBytes, "a warp's place");

__device__ __forceinline__ void store_row16(void* out, int dtype, int64_t at, const float* v) {  // 16 elements
  if (dtype == SPHKV_F32) {
    float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    return;
  }
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (dtype == SPHKV_BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      w[i] = pack_f16x2(v[2 * i], v[2 * i + 1]);
    }
  }
  uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + at);
  o[0] = make_uint4(w[0], w[1], w[2], w[3]);
  o[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

template <int DH, bool I8>
__global__ void __launch_bounds__(kAtThreads, 1) blocks_attend_kernel(const __grid_constant__ AtArgs a) {
  using L = At<DH>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t base = smem_u32(smem), bars = base + L::kBars;
  AtMeta* const metas = reinterpret_cast<AtMeta*>(smem + L::kMeta);
  __shared__ uint32_t tmem_at;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + 8 * (kNext + i), 9), mbar_init(bars + 8 * (kKFree + i), 1);
      mbar_init(bars + 8 * (kVFull + i), 4), mbar_init(bars + 8 * (kVFree + i), 1);
      mbar_init(bars + 8 * (kQFull + i), 4), mbar_init(bars + 8 * (kSFull + i), 1);
      mbar_init(bars + 8 * (kPFull + i), 4), mbar_init(bars + 8 * (kODone + i), 1);
    }
    mbar_init(bars + 8 * kLast, 1);
    fence_async_smem();
  }
  if (warp == kAtProducts) tmem_alloc(smem_u32(&tmem_at), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  griddep_wait();
  const uint32_t* prefix = a.prefix;
  const AtItem* items = a.items;
  if (prefix == nullptr) {
    uint32_t* const at = reinterpret_cast<uint32_t*>(smem + L::kPrefix);
    AtItem* const of = reinterpret_cast<AtItem*>(smem + L::kItems);
    deal_tiles(a.slots, at, of, [&](int s) { return item_of(a, s); });
    prefix = at;
    items = of;
  }
  AtWalk& walk = *reinterpret_cast<AtWalk*>(smem + L::kWalks + warp * kAtWalkBytes);
  const AtItem& u = walk.u;
  if (lane == 0) {
    walk.prefix = prefix;
    walk.items = items;
    walk.begin(a, blockIdx.x);
  }
  bool lost = false;
  auto wait = [&](int bar, uint32_t n) {  // the n-th phase, from 0
    if (!lost && !mbar_wait(bars + 8 * bar, n & 1)) {
      lost = true;
      bad_status(a.c, SPHKV_ST_TIMEOUT);
    }
    return !lost;
  };
  auto warp_wait = [&](int bar, uint32_t n) { return __all_sync(0xffffffffu, wait(bar, n)); };
  auto next_segment = [&] {
    __syncwarp();  // the segment before has been read
    const int more = lane == 0 ? walk.next(a) : 0;
    __syncwarp();  // what lane 0 wrote is there for all: a shuffle alone orders no memory
    return __shfl_sync(0xffffffffu, more, 0) != 0;
  };

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax
    regs_up<kAtRegsSoftmax>();
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;  // of the tile
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t s_at = tmem + lanes + t * 128, o_at = tmem + lanes + 256 + t * 128;
    const float kNone = -3.402823466e38f;
    uint32_t tile = 0, taken = 0, segs = 0;  // key tiles of the worker; those with this row tile; segments with it
    while (!lost && next_segment()) {
      const int cnt = walk.cnt[t], flat = 128 * t + row;
      float m = kNone, l = 0.f, big = 0.f;
      if (cnt > 0) {
        const bool live = flat < u.rows;
        const int lim = live ? u.pos0 + (u.r0 + flat) / a.group + 1 : u.lim[t], first = u.first;
        const int least = u.pos0 + (u.r0 + 128 * t) / a.group + 1;  // of the tile's rows
        const int seg_key0 = (u.kt0 + walk.from) * kAtKeys;
        // The warp's 32 rows of queries, scaled by powers of two into f16: DH / 8 lanes to a row.
        constexpr int LPR = DH / 8, RPL = 32 / LPR, NQ = 32 / RPL;
        const int tok0 = u.r0 / a.group, rem0 = u.r0 - tok0 * a.group;
        const uint32_t per_group = 65535u / a.group + 1u;  // x / group = x * per_group >> 16 for x below 2^13
        const bool bf = a.q_dtype == SPHKV_BF16;
        const uint32_t q_at = base + L::kQ + t * L::kOperand;
        uint32_t mine = 0;  // the largest magnitude of this thread's row, as bits
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
          uint4 raw[NQ / 2];
#pragma unroll
          for (int i = 0; i < NQ / 2; ++i) {
            const int r = 128 * t + 32 * (warp & 3) + RPL * (i + part * (NQ / 2)) + lane / LPR;
            const uint32_t of = rem0 + min(r, u.rows - 1), tk = of * per_group >> 16;  // rows behind the last are its like, and are not written
            const uint16_t* const src = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(u.row0 + tok0 + (int)tk) * a.q_row_stride +
                                        (int64_t)(walk.head * a.group + (int)(of - tk * a.group)) * a.q_head_stride + 8 * (lane % LPR);
            if (a.q_vec) {
              raw[i] = *reinterpret_cast<const uint4*>(src);
            } else {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = (uint32_t)src[2 * k] | ((uint32_t)src[2 * k + 1] << 16);
              raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
#pragma unroll
          for (int i = 0; i < NQ / 2; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
#pragma unroll
            for (int x = 1; x < LPR; x <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, x));
            const uint32_t th = max(top >> 16, top & 0xffffu);
            const uint16_t th16 = (uint16_t)th;
            const uint32_t tb = bf ? th << 16 : __float_as_uint(__half2float(*reinterpret_cast<const __half*>(&th16)));
            const int r = RPL * (i + part * (NQ / 2));  // of the warp's
            const uint32_t theirs = __shfl_sync(0xffffffffu, tb, (lane % RPL) * LPR);
            if (lane / RPL == r / RPL) mine = theirs;
            int e = (int)(tb >> 23);
            e = e == 255 ? 140 : max(e, 14);
            const float sc = __uint_as_float(((uint32_t)(267 - e) << 23) | a.q_sign);
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float2 x;
              if (bf)
                x = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
              else
                x = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
              h[k] = pack_f16x2(x.x * sc, x.y * sc);
            }
            sts_u4(q_at + operand_at(32 * (warp & 3) + r + lane / LPR, lane % LPR), h[0], h[1], h[2], h[3]);
          }
        }
        int e = (int)(mine >> 23);
        e = e == 255 ? 140 : max(e, 14);
        const float f = __uint_as_float((uint32_t)(e - 13) << 23) * a.scale_log2;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + 8 * (kQFull + t));

        for (int k = 0; k < cnt; ++k) {
          const uint32_t n = tile + k;
          // the products' warp saw the tile's scales before it asked for the logits
          if (!warp_wait(kSFull + t, taken)) break;
          ++taken;
          tc_fence_after();
          const uint32_t meta_at = base + L::kMeta + (n & 3) * (uint32_t)sizeof(AtMeta);  // read anew in every pass: kept, 32 registers would not be there for logits
          const int key0 = seg_key0 + k * kAtKeys;
          const float4 tail = lds_f4(meta_at + 128);
          const float down = tail.x;
          big = tail.y;
          const uint32_t bad = __float_as_uint(tail.z);
          const bool edge = key0 < first || key0 + kAtKeys > least || bad != 0;  // the same for all rows of the tile
          // The row's reference moves to `to` in front of 32 keys: sums, outputs (with `down`: the value scales' reference) and
          // the weights of the tile's keys before them follow.
          auto move = [&](float to, float by, int done) {
            const float d = ex2(m - to);
            m = to;
            l *= d;
            if (k > 0) {  // O holds something
              const float r = d * by;
#pragma unroll 1
              for (int i = 0; i < DH / 16; ++i) {
                float o[16];
                tmem_ld_x16(o_at + 16 * i, o);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 16; ++c) o[c] *= r;
                tmem_st_x16(o_at + 16 * i, o);
              }
            }
            // References are whole numbers, so d is a power of two and weights stay rounded once, but for what falls below f16's normal
            // numbers: 2^-25.  Two factors, as d itself may lie there (one product in fp32: 104.6 us for the five pieces instead of 102.8).
            const float most = fmaxf(d, 0x1p-14f), rest = fminf(d * 0x1p14f, 1.f);
            const uint32_t d1 = pack_f16x2(most, most), d2 = pack_f16x2(rest, rest);
            tmem_wait_st();
#pragma unroll 1
            for (int h = 0; h < done; ++h) {
              float w[16];
              tmem_ld_x16(s_at + 16 * h, w);
              tmem_wait_ld();
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const uint32_t v = __float_as_uint(w[c]);
                const __half2 r = __hmul2(__hmul2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&d1)),
                                          *reinterpret_cast<const __half2*>(&d2));
                w[c] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&r));
              }
              tmem_st_x16(s_at + 16 * h, w);
            }
            tmem_wait_st();  // an odd group of 16 keys stores its weights into the last of these columns
          };
          if (down != 1.f) {
            // S has grown.  The row's reference goes the other way, so that O stays as it is; where the sum would grow past
            // 32 bits (or all scales were 0) O shrinks instead, row by row.
            const int e = (int)(__float_as_uint(down) >> 23) - 127;  // a power of two
            const float grown = l * __uint_as_float((uint32_t)(127 - max(e, -80)) << 23);
            const bool stays = e >= -80 && !(grown > 0x1p110f);
            if (__any_sync(0xffffffffu, !stays)) move(m, stays ? 1.f : down, 0);
            if (stays) {
              m += (float)e;
              l = grown;
            }
          }
          if (edge) {
#pragma unroll 1
            for (int g = 0; g < 8; ++g) {
              float v[16];
              tmem_ld_x16(s_at + 16 * g, v);
              tmem_wait_ld();
              const float4 of = lds_f4(meta_at + 16 * g);
              float top = -INFINITY;
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                if (key0 + 16 * g + c < first || key0 + 16 * g + c >= lim || ((bad >> g) & 1)) v[c] = -INFINITY;
                top = fmaxf(top, v[c]);
              }
              top = fmaf(top, of.x * f, of.y);
              const bool up = top > m + kAtLazy;
              // 16 keys are half of what move() counts in: an odd group's first half has not been stored yet
              if (__any_sync(0xffffffffu, up)) move(up ? ceilf(top - kAtWeight) : m, 1.f, (g + 1) >> 1);
              float all = 0.f;
              uint32_t p[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {  // scales may be zero or NaN where nothing is seen
                const float y = v[2 * i], z = v[2 * i + 1];
                const float e = y == -INFINITY ? 0.f : ex2(fmaf(y, of.x * f, of.y - m)), h = z == -INFINITY ? 0.f : ex2(fmaf(z, of.x * f, of.y - m));
                all += e + h;
                p[i] = (bad >> (8 + g)) & 1 ? 0u : pack_f16x2(e, h);  // their values count as zeros
              }
              l += all == 0.f ? 0.f : all * of.z;
              tmem_st_x8u(s_at + 8 * g, p);  // over logits that have been read
              tmem_wait_st();
            }
          } else {
            // 32 keys at a time, in a loop that stays one: with all 128 in sight the compiler starts more than it has registers
            // for.  The next 32 travel while the first half of the exponentials is taken, and their largest is found beside the
            // second half (behind the last 32 the first are read again, to no purpose: a branch would part the two).
            float x[32], mx;
            float4 of[2];
            auto highest = [&] {
              float top[2];
#pragma unroll
              for (int gg = 0; gg < 2; ++gg) {
                const float* const v = x + 16 * gg;
                float even = fmaxf(fmaxf(v[0], v[1]), v[2]), odd = fmaxf(fmaxf(v[3], v[4]), v[5]);
#pragma unroll
                for (int i = 6; i < 14; i += 4) even = fmaxf(fmaxf(even, v[i]), v[i + 1]), odd = fmaxf(fmaxf(odd, v[i + 2]), v[i + 3]);
                top[gg] = fmaf(fmaxf(fmaxf(fmaxf(even, v[14]), v[15]), odd), of[gg].x * f, of[gg].y);
              }
              mx = fmaxf(top[0], top[1]);
            };
            of[0] = lds_f4(meta_at), of[1] = lds_f4(meta_at + 16);
            tmem_ld_x32(s_at, x);
            tmem_wait_ld();
            highest();
#pragma unroll 1
            for (int h = 0; h < 4; ++h) {
              const bool up = mx > m + kAtLazy;
              if (__any_sync(0xffffffffu, up)) move(up ? ceilf(mx - kAtWeight) : m, 1.f, h);
              float2 e[16], part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
              uint32_t p[16];
#pragma unroll
              for (int gg = 0; gg < 2; ++gg) {
                const float c = of[gg].x * f, add = of[gg].y - m;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  e[8 * gg + i] = __ffma2_rn(make_float2(x[16 * gg + 2 * i], x[16 * gg + 2 * i + 1]), make_float2(c, c), make_float2(add, add));
              }
              const float up0 = of[0].z, up1 = of[1].z;
              const int next = (h + 1) & 3;
              of[0] = lds_f4(meta_at + 32 * next), of[1] = lds_f4(meta_at + 32 * next + 16);
              tmem_ld_x32(s_at + 32 * next, x);
              auto weigh = [&](int i) {
                if ((i & 7) == 1)  // an eighth: 1.12 ms, none 1.13, a quarter 1.13, three eighths 1.15, half 1.19
                  e[i] = ex2_poly(e[i]);
                else
                  e[i].x = ex2(e[i].x), e[i].y = ex2(e[i].y);
                part[i >> 3] = __fadd2_rn(part[i >> 3], e[i]);
                p[i] = pack_f16x2(e[i].x, e[i].y);
              };
#pragma unroll
              for (int i = 0; i < 8; ++i) weigh(i);
              tmem_wait_ld();
#pragma unroll
              for (int i = 8; i < 16; ++i) weigh(i);
              highest();
              l += (part[0].x + part[0].y) * up0;
              l += (part[1].x + part[1].y) * up1;
              tmem_st_x16u(s_at + 16 * h, p);  // over logits that have been read
            }
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + 8 * (kPFull + t));
        }
        if (!lost) (void)warp_wait(kODone + t, segs);
        lost = __any_sync(0xffffffffu, lost);
        ++segs;
      }
      tile += walk.count;
      if (lost) break;
      // ---- the segment's outputs ----
      if (128 * t < u.rows) {
        const bool live = flat < u.rows;
        const int tok = (u.r0 + flat) / a.group, hd = walk.head * a.group + (u.r0 + flat) - tok * a.group;
        const int64_t dense = (int64_t)u.row0 + tok;
        const float scale = big * 0x1p-6f;  // of outputs and sums of a part
        float* const part = a.parts + ((int64_t)blockIdx.x * 2 + (walk.from > 0 ? 0 : 1)) * (DH + 2) * kAtRows + flat;
        const float per = l == 0.f ? 0.f : big / l;
        tc_fence_after();
#pragma unroll 1
        for (int i = 0; i < DH / 16; ++i) {
          float o[16];
          __syncwarp();
          if (cnt > 0) {
            tmem_ld_x16(o_at + 16 * i, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = 0.f;
          }
          if (live && walk.whole) {
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = l == 0.f ? 0.f : o[c] * per;
            store_row16(a.out, a.out_dtype, (dense * a.Hq + hd) * DH + 16 * i, o);
          } else if (live) {
#pragma unroll
            for (int c = 0; c < 16; ++c) part[(2 + 16 * i + c) * kAtRows] = o[c] * scale;
          }
        }
        if (live && !walk.whole) part[0] = l == 0.f ? -INFINITY : m, part[kAtRows] = l * 0x1p-6f;
        tc_fence_before();
      }
    }
  } else if (warp < kAtProducts) {
    // ---------------------------------------------------------------- codes to operands: four warps for keys, four for values
    regs_down<kAtRegsCodes>();
    constexpr int NL = DH / 16, TPL = 512 / DH;  // loads of a lane; tokens of a load
    const bool values = warp >= 12;
    const int w = warp & 3;
    // a quarter warp stores 16-byte chunks of two rows that differ in the swizzle's last bit: no bank twice
    const int ts = DH == 128 ? ((lane >> 2) & 1) + 2 * (lane >> 4) : lane >> 2;
    const int ch = DH == 128 ? (lane & 3) + 4 * ((lane >> 3) & 1) : lane & 3;
    const int shift = 31 - __clz(a.c.page_size);
    const uint8_t* const codes = reinterpret_cast<const uint8_t*>(values ? a.c.v_codes : a.c.k_codes) + ts * DH + 16 * ch;
    const int full = values ? kVFull : kNext, free = values ? kVFree : kKFree;
    const uint32_t to = base + (values ? L::kV : L::kK);
    uint32_t n = 0;  // key tiles of the worker
    if (values && lane == 0) mbar_arrive(bars + 8 * kNext);  // no values before the first tile
    while (!lost && next_segment()) {
      const int limit = max(u.lim[0], u.lim[1]), key_begin = (u.kt0 + walk.from) * kAtKeys;
      const int32_t* table = a.c.block_table + (int64_t)u.b * a.c.max_blocks;
      // lanes 0 .. 7 look after a tile's eight groups of 16 keys
      auto page_of = [&](int k) {
        const int t0 = key_begin + k * kAtKeys + 16 * (lane & 7);
        return k < walk.count && t0 < limit && t0 + 16 > u.first ? table[t0 >> shift] : -2;
      };
      auto checked = [&](int page) {
        if (page == -2) return -2;  // before the keys, or behind them: the table need not name a page
        if (page < 0 || page >= a.c.n_pages) {
          bad_status(a.c, SPHKV_ST_BAD_BLOCK);
          return -1;
        }
        return page;
      };
      // Every load is made, from a row that exists: a load that may be skipped ends in a copy that waits for it.
      uint4 raw[NL];
      auto load = [&](int k, int page) {
        const int at_row = page >= 0 ? ((page * a.c.Hkv + walk.head) << shift) + ((key_begin + k * kAtKeys + 16 * (lane & 7)) & (a.c.page_size - 1)) : 0;
        const uint8_t* const at[2] = {codes + (int64_t)__shfl_sync(0xffffffffu, at_row, 2 * w) * DH,
                                      codes + (int64_t)__shfl_sync(0xffffffffu, at_row, 2 * w + 1) * DH};
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const float4 v = ldg_stream_f4(at[TPL * i / 16] + (TPL * i & 15) * DH);
          raw[i] = make_uint4(__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w));
        }
      };
      int page = checked(page_of(0)), next_page = page_of(1);
      load(0, page);
      for (int k = 0; k < walk.count; ++k, ++n) {
        const uint32_t st = n & 1;
        const int now = page;
        if (n >= 2 && !warp_wait(free + st, (n >> 1) - 1)) break;
        const int warp_key0 = key_begin + k * kAtKeys + 32 * w, there = limit - warp_key0, before = u.first - warp_key0;
        if (there < 32 || before > 0 || __any_sync(0xffffffffu, now < 0)) {  // rows that are no keys', or of no page, may be any bytes
#pragma unroll
          for (int i = 0; i < NL; ++i) {
            const int its = __shfl_sync(0xffffffffu, now, 2 * w + (TPL * i) / 16);
            if (TPL * i + ts >= there || TPL * i + ts < before || its < 0) raw[i] = make_uint4(0, 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const uint32_t c[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          uint32_t h[8];
#pragma unroll
          for (int q = 0; q < 4; ++q) codes_to_f16<I8>(c[q], h[2 * q], h[2 * q + 1]);
          const uint32_t place = to + st * L::kOperand;
          const int t = 32 * w + TPL * i + ts;
          sts_u4(place + operand_at(t, 2 * ch), h[0], h[1], h[2], h[3]);
          sts_u4(place + operand_at(t, 2 * ch + 1), h[4], h[5], h[6], h[7]);
        }
        fence_async_smem();
        __syncwarp();
        // Behind a segment's last tile values are asked for ahead of the next step's keys: their second tile may not count for the
        // step before it.
        if (values && n >= 1 && !warp_wait(kNext + (st ^ 1), (n - 1) >> 1)) break;
        if (lane == 0) {
          mbar_arrive(bars + 8 * (full + st));
          if (values) mbar_arrive(bars + 8 * (kNext + (st ^ 1)));
        }
        // the next tile's codes are asked for as soon as their registers are free
        page = checked(next_page);
        next_page = page_of(k + 2);
        if (k + 1 < walk.count) load(k + 1, page);
      }
      lost = __any_sync(0xffffffffu, lost);
    }
  } else {
    regs_down<kAtRegsRest>();
    if (warp == kAtProducts) {
      // -------------------------------------------------------------- products
      constexpr uint32_t kIdescS = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
      constexpr uint32_t kIdescO = (1u << 4) | (((uint32_t)DH >> 3) << 17) | ((128u >> 4) << 24) | (1u << 16);
      // descriptors: what is constant above the address bits, and addresses in units of 16 bytes
      const uint64_t rows_of_64 = smem_desc(0, 0, 1024, 2), values_of = smem_desc(0, DH == 128 ? L::kSlab : 0, 1024, 2);
      const uint32_t unit = base >> 4;
      uint32_t n = 0, p_phase = 0, q_phase = 0;  // bit t: the phase that row tile t's barrier is in
      auto phase_wait = [&](int bar, uint32_t& phases, int t) {
        const bool ok = warp_wait(bar + t, phases >> t);
        phases ^= 1u << t;
        return ok;
      };
      // the whole warp waits, one elected thread issues: under a condition on the lane the compiler does not see that it is one
      bool issued = false;
      while (!lost && next_segment()) {
        const int count = walk.count;
#pragma unroll 1
        for (int t = 0; t < 2; ++t)
          if (walk.cnt[t] > 0 && !phase_wait(kQFull, q_phase, t)) break;
#pragma unroll 1
        for (int k = 0; k <= count; ++k) {
          const uint32_t st = (n + k) & 1, before = st ^ 1;
          if (!(k < count ? warp_wait(kNext + st, (n + k) >> 1) : warp_wait(kVFull + before, (n + k - 1) >> 1))) break;
          bool ok = true;
#pragma unroll 1
          for (int t = 0; t < 2; ++t) {
            const int cnt = walk.cnt[t];
            if (ok && k > 0 && k <= cnt) {
              ok = phase_wait(kPFull, p_phase, t);
              tc_fence_after();
              if (ok && elect_one()) {
                const uint64_t v_desc = values_of | (unit + ((L::kV + before * L::kOperand) >> 4));
#pragma unroll
                for (int i = 0; i < kAtKeys / 16; ++i)
                  mma_ts(tmem + 256 + t * 128, tmem + t * 128 + 8 * i, v_desc + (uint64_t)((i * 2048) >> 4), kIdescO, k > 1 || i > 0);
                if (k == cnt) mma_commit(bars + 8 * (kODone + t));
              }
              __syncwarp();
            }
            if (ok && k < cnt) {
              tc_fence_after();
              if (elect_one()) {
                const uint64_t q_desc = rows_of_64 | (unit + ((L::kQ + t * L::kOperand) >> 4));
                const uint64_t k_desc = rows_of_64 | (unit + ((L::kK + st * L::kOperand) >> 4));
#pragma unroll
                for (int i = 0; i < DH / 16; ++i) {
                  const uint64_t step = (uint64_t)(((i >> 2) * L::kSlab + (i & 3) * 32) >> 4);
                  mma_ss(tmem + t * 128, q_desc + step, k_desc + step, kIdescS, i > 0);
                }
                mma_commit(bars + 8 * (kSFull + t));
              }
              __syncwarp();
              issued = true;
            }
          }
          if (!ok) break;
          if (elect_one()) {
            if (k < count) mma_commit(bars + 8 * (kKFree + st));
            if (k > 0) mma_commit(bars + 8 * (kVFree + before));
          }
          __syncwarp();
        }
        lost = __any_sync(0xffffffffu, lost);
        n += count;
      }
      if (issued) {  // nothing may be on its way when tensor and shared memory are given back
        if (elect_one()) mma_commit(bars + 8 * kLast);
        __syncwarp();
        (void)mbar_wait(bars + 8 * kLast, 0);
      }
    } else if (warp == kAtProducts + 1) {
      // -------------------------------------------------------------- scales of the key tiles, for the softmax
      const int shift = 31 - __clz(a.c.page_size);
      uint32_t n = 0;
      while (!lost && next_segment()) {
        const int limit = max(u.lim[0], u.lim[1]), key_begin = (u.kt0 + walk.from) * kAtKeys + 16 * (lane & 7);
        const int32_t* table = a.c.block_table + (int64_t)u.b * a.c.max_blocks;
        auto page_of = [&](int k) {
          const int t0 = key_begin + k * kAtKeys;
          return k < walk.count && t0 < limit && t0 + 16 > u.first ? table[t0 >> shift] : -2;
        };
        auto scale_of = [&](const float* scales, int page) {
          return page >= 0 && page < a.c.n_pages ? scales[page * a.c.Hkv + walk.head] : 0.f;
        };
        int page = page_of(0), next_page = page_of(1);
        float big = 0.f, ks = scale_of(a.c.k_scale, page), vs = scale_of(a.c.v_scale, page);
        for (int k = 0; k < walk.count; ++k, ++n) {
          const bool there = page >= 0 && page < a.c.n_pages;
          const float ks_now = ks, vs_now = vs;
          unsigned bad = __ballot_sync(0xffffffffu, page != -2 && !there) & 0xffu;
          page = next_page;
          next_page = page_of(k + 2);
          ks = scale_of(a.c.k_scale, page), vs = scale_of(a.c.v_scale, page);
          float top = vs_now < INFINITY ? vs_now : 0.f;  // rows that do not see a page without a scale keep theirs
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          float down = 1.f;
          if (top > big) {
            const float b = __uint_as_float(min((__float_as_uint(top) + 0x7fffffu) & 0x7f800000u, 0x7e800000u));
            down = big > 0.f ? big / b : 0.f;
            big = b;
          }
          const float ref = big > 0.f ? big : 1.f;
          // The sum of weights takes v out again, which 32 bits allow down to 2^-80: values that are smaller still count as zeros,
          // like those of scale 0.  Theirs is the smallest v, so that they do not raise a row's reference above what it sees of others.
          float v = vs_now * (1.f / ref);
          const bool zeros = v < 0x1p-80f;
          if (zeros) v = 0x1p-80f;
          bad |= (__ballot_sync(0xffffffffu, there && zeros) & 0xffu) << 8;
          // as far ahead as keys may be: the softmax has left tile n - 3 behind, and this place held n - 4
          if (n >= 2 && !warp_wait(kKFree + (n & 1), (n >> 1) - 1)) break;
          AtMeta& mt = metas[n & 3];
          if (lane < 8) mt.of[lane] = make_float4(ks_now, log2f(v), 1.f / v, 0.f);
          if (lane == 0) mt.down = k == 0 ? 1.f : down, mt.big = ref, mt.bad = bad;
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + 8 * (kNext + (n & 1)));
        }
        lost = __any_sync(0xffffffffu, lost);
      }
    } else if (warp == kAtProducts + 2) {
      // -------------------------------------------------------------- what the second launch joins; queries that see nothing
      if (lane == 0) {
        const Shares shares(prefix[a.slots] * a.c.Hkv, a.workers);
        AtSpan span = {};
        if (blockIdx.x < shares.n) {
          const uint32_t stop = shares.start(blockIdx.x + 1);
          const int slot = slot_at(prefix, a.slots, (stop - 1) / a.c.Hkv);
          const AtItem it = items[slot];
          span.head = (stop - 1 - prefix[slot] * a.c.Hkv) / (uint32_t)it.tiles;
          const uint32_t p0 = prefix[slot] * a.c.Hkv + span.head * it.tiles, end = p0 + it.tiles;
          if (p0 >= shares.start(blockIdx.x) && end > stop) span.n = shares.owner(end - 1) - blockIdx.x + 1;
          span.row0 = it.row0, span.r0 = it.r0, span.rows = it.rows;
        }
        a.spans[blockIdx.x] = span;
      }
#pragma unroll 1
      for (int s = blockIdx.x; s < a.slots; s += gridDim.x) {
        if (prefix[s + 1] != prefix[s]) continue;
        const AtItem it = items[s];
        const float none[16] = {};
#pragma unroll 1
        for (int r = lane; r < it.rows; r += 32) {
          const int tok = (it.r0 + r) / a.group, g = it.r0 + r - tok * a.group;
#pragma unroll 1
          for (int i = 0; i < a.c.Hkv * (DH / 16); ++i)
            store_row16(a.out, a.out_dtype, ((int64_t)(it.row0 + tok) * a.Hq + i / (DH / 16) * a.group + g) * DH + 16 * (i % (DH / 16)), none);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kAtProducts) tmem_dealloc(tmem, 512);
}

// CTA (w, y): the block that worker w begins and others go on with, dims 16 y .. of it.
__global__ void __launch_bounds__(256) blocks_attend_merge_kernel(const __grid_constant__ AtArgs a, int dh) {
  griddep_launch();
  const int flat = threadIdx.x, w = blockIdx.x, d0 = 16 * blockIdx.y;
  const AtSpan u = a.spans[w];
  if (u.n == 0 || flat >= u.rows) return;
  const int n = u.n, head = u.head;
  const int size = (dh + 2) * kAtRows;
  float o[16];
#pragma unroll
  for (int c = 0; c < 16; ++c) o[c] = 0.f;
  float top = -INFINITY, sum = 0.f;
  const float* const mine = a.parts + ((int64_t)2 * w + 1) * size + flat;  // the others' are their first places
  auto part = [&](int x) { return x == 0 ? mine : mine + (int64_t)(2 * x - 1) * size; };
#pragma unroll 4
  for (int x = 0; x < n; ++x) top = fmaxf(top, part(x)[0]);
#pragma unroll 2
  for (int x = 0; x < n; ++x) {
    const float* const p = part(x);
    const float f = p[0] == -INFINITY ? 0.f : ex2(p[0] - top);  // nothing seen there: its outputs are zeros
    sum += p[kAtRows] * f;
#pragma unroll
    for (int c = 0; c < 16; ++c) o[c] += p[(2 + d0 + c) * kAtRows] * f;
  }
#pragma unroll
  for (int c = 0; c < 16; ++c) o[c] = sum == 0.f ? 0.f : o[c] / sum;
  const int tok = (u.r0 + flat) / a.group, hd = head * a.group + u.r0 + flat - tok * a.group;
  store_row16(a.out, a.out_dtype, ((int64_t)(u.row0 + tok) * a.Hq + hd) * dh + d0, o);
}

static int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
static int64_t at_slots(int64_t rows, int B, int group) { return (rows * group >> 8) + B; }  // at least block_slots()
static int64_t at_scratch(int64_t rows, int B, int group, int dh, int sms) {
  return align256((at_slots(rows, B, group) + 1) * 4) + align256(at_slots(rows, B, group) * (int64_t)sizeof(AtItem)) + align256(sms * (int64_t)sizeof(AtSpan)) + (int64_t)sms * 2 * (dh + 2) * kAtRows * 4;
}

template <int DH, bool I8>
static int launch_at(const AtArgs& a, cudaStream_t st) {
  static SmemOptIn opt_in;
  auto kern = blocks_attend_kernel<DH, I8>;
  if (int rc = ensure_dynamic_smem(opt_in, (const void*)kern, At<DH>::kSmem, "blocks_attend")) return rc;
  // a launch with fewer registers could not hand out what the softmax asks for, and would wait for them
  static const int regs = [&] {
    cudaFuncAttributes f;
    return cudaFuncGetAttributes(&f, (const void*)kern) == cudaSuccess ? f.numRegs : -1;
  }();
  SPHKV_REQUIRE(regs == kAtRegs, SPHKV_E_LIMIT, "blocks_attend: compiled for %d registers, needs %d", regs, kAtRegs);
  (void)launch_overlapped(kern, dim3(a.workers), dim3(kAtThreads), At<DH>::kSmem, st, a);
  return check_launch("blocks_attend_kernel");
}

// One sequence's tokens in the decode kernel's eight rows: there the codes are not turned into operands in shared memory.
static bool few_rows(const BlockRows& r, int B, int group) { return r.rows <= (int64_t)B << tokens_shift(group); }

}  // namespace sphkv

using namespace sphkv;

extern "C" int64_t sphkv_blocks_attend_scratch_bytes(int32_t B, int64_t rows, int32_t Hq, int32_t Hkv, int32_t dh) {
  if (B <= 0 || rows < 0 || rows > 0x7ffffff || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > SPHKV_MAX_GQA || (dh != 64 && dh != 128))
    return SPHKV_E_ARG;
  const int sms = sm_count_current_device();
  if (sms <= 0) return sms;
  const int group = Hq / Hkv;
  const int64_t many = at_scratch(rows, B, group, dh, sms);
  const BlockRows r = {nullptr, (int)rows, 0, 1, false};
  return few_rows(r, B, group) ? max(many, few_queries_scratch(rows, B, Hkv, dh, tokens_shift(group), sms)) : many;
}

extern "C" int sphkv_blocks_attend(const sphkv_blocks* c, const void* q, int32_t q_dtype, int64_t q_row_stride, int64_t q_head_stride,
                                   const int32_t* cu, int64_t rows, const int32_t* first, void* out, int32_t out_dtype, void* scratch,
                                   int64_t scratch_bytes, int32_t Hq, float sm_scale, void* stream) {
  if (int rc = check_blocks(c, "blocks_attend")) return rc;
  AtArgs a = {};
  a.c = *c;
  if (int rc = block_rows(a.r, c, cu, rows, "blocks_attend")) return rc;
  SPHKV_REQUIRE(rows <= 0x7ffffff, SPHKV_E_LIMIT, "blocks_attend: rows=%lld (max 2^27 - 1)", (long long)rows);
  if (rows == 0) return 0;  // tensors without elements have no address
  SPHKV_REQUIRE(q != nullptr, SPHKV_E_ARG, "blocks_attend: q is NULL");
  if (int rc = check_queries(*c, q, q_dtype, out, nullptr, out_dtype, Hq, sm_scale, "blocks_attend")) return rc;
  SPHKV_REQUIRE(q_dtype != SPHKV_F32, SPHKV_E_DTYPE, "blocks_attend: q_dtype=%d (16-bit types)", q_dtype);
  SPHKV_REQUIRE(((uintptr_t)out & 15) == 0, SPHKV_E_ALIGN, "blocks_attend: out needs 16 B");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int group = Hq / c->Hkv, sms = sm_count_current_device();
  if (sms <= 0) return sms;
  if (few_rows(a.r, c->B, group))
    return few_queries(*c, a.r, q, q_dtype, q_row_stride, q_head_stride, first, out, out_dtype, nullptr, scratch, scratch_bytes, Hq, sm_scale,
                       tokens_shift(group), "blocks_attend", st);
  a.r.mul = group;
  a.q = q;
  a.q_dtype = q_dtype;
  a.q_row_stride = q_row_stride;
  a.q_head_stride = q_head_stride;
  a.q_vec = ((uintptr_t)q & 15) == 0 && (((q_row_stride | q_head_stride) * 2) & 15) == 0;
  a.first = first;
  a.out = out;
  a.out_dtype = out_dtype;
  a.Hq = Hq;
  a.group = group;
  a.q_sign = sm_scale < 0.f ? 0x80000000u : 0u;
  a.scale_log2 = fabsf(sm_scale) * kLog2e;
  a.workers = sms;
  const int64_t slots = block_slots(a.r, c->B, 8, 1);
  // key tiles of all blocks of queries are counted in 32 bits
  SPHKV_REQUIRE((double)slots * c->Hkv * ((int64_t)c->max_blocks * c->page_size / kAtKeys + 2) < 2147483648.0, SPHKV_E_LIMIT,
                "blocks_attend: too many (query block, head, token)s for one launch");
  a.slots = (int)slots;
  const int64_t need = at_scratch(rows, c->B, group, c->dh, sms);
  SPHKV_REQUIRE(scratch != nullptr && scratch_bytes >= need, SPHKV_E_SCRATCH, "blocks_attend: scratch %lld B < %lld B",
                (long long)scratch_bytes, (long long)need);
  SPHKV_REQUIRE(((uintptr_t)scratch & 255) == 0, SPHKV_E_ALIGN, "blocks_attend: scratch needs 256 B");
  uint8_t* const items_at = reinterpret_cast<uint8_t*>(scratch) + align256((at_slots(rows, c->B, group) + 1) * 4);
  a.spans = reinterpret_cast<AtSpan*>(items_at + align256(at_slots(rows, c->B, group) * (int64_t)sizeof(AtItem)));
  a.parts = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.spans) + align256(sms * (int64_t)sizeof(AtSpan)));
  if (slots > kDealt) {
    uint32_t* const prefix = reinterpret_cast<uint32_t*>(scratch);
    AtItem* const items = reinterpret_cast<AtItem*>(items_at);
    (void)launch_overlapped(blocks_attend_plan_kernel, dim3(1), dim3(1024), 0, st, a, prefix, items);
    if (int rc = check_launch("blocks_attend_plan_kernel")) return rc;
    a.prefix = prefix;
    a.items = items;
  }
  const bool i8 = c->store == SPHKV_BLOCKS_I8;
  const int rc = c->dh == 128 ? (i8 ? launch_at<128, true>(a, st) : launch_at<128, false>(a, st))
                              : (i8 ? launch_at<64, true>(a, st) : launch_at<64, false>(a, st));
  if (rc) return rc;
  blocks_attend_merge_kernel<<<dim3(a.workers, c->dh / 16), 256, 0, st>>>(a, c->dh);
  return check_launch("blocks_attend_merge_kernel");
}
