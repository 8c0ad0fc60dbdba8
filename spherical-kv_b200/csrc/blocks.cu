// The 8-bit block cache: quantising tokens as they are written, and reading them back.
//
// Both move bytes: a bf16 token of 8 heads of 128 dims is 4096 bytes to read and 2048 to write, and the other way round.  A warp has 16
// slots of one (page, side, head), so a page of 16 tokens needs no barrier; the largest magnitude and the rounding work on the
// same registers, so tokens are read once.  Measured (32768 bf16 tokens, 16-token pages, int8, cold caches): append 47 us where
// the bytes take 31 at the copy rate, bound by instructions (16.4 an element, 70 % of issue slots at 43 % of the warps; 64 registers a thread give
// four blocks an SM, 5 % faster than three); read 34 us, as long as the bytes take.  Steps of one token are latency: 3 us each.
#include <type_traits>

#include "blocks.cuh"

namespace sphkv {

struct BlocksIo {
  sphkv_blocks c;
  BlockRows r;
  const void* src[2];  // keys, values (append)
  void* dst[2];        // (read)
  int64_t row_stride[2], head_stride[2];
  int slots, shift;  // page_size = 1 << shift
  bool vec;          // rows on 16-byte boundaries
};

constexpr int kIoThreads = 256;  // eight warps, each with 16 tokens of one (page, side, head)
constexpr float kLeastScale = 0x1p-110f, kLift = 0x1p64f;  // scale times border has a last bit of 2^-33 of the scale, and fp32 ends at 2^-149
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds |q| < 2^22 to a whole number, ties to even

// ---- nearest 8-bit codes -----------------------------------------------------------------------------------
// q approximates the quotient to 1.5 ulp (a rounded reciprocal or ratio, one product).  Where that leaves the nearest code
// open, within 2^-15 of a whole number's border or 4 ulp of an e4m3 border, the sign of x - border * s decides, which one fma gives
// exactly: a border has 8 bits at most, the product 32, and a rounding keeps the sign of what is not below fp32's least number (so
// the smallest scales and their tokens are multiplied by a power of two first).  bf16 tokens lie exactly on borders often, since scale
// and token are quotients of 8-bit numbers: some word of most rows is open, and 64-bit division there was half of the kernel's
// instructions.
template <bool I8>
__device__ uint32_t code_of_double(double q) {
  if constexpr (I8) return (uint32_t)(int)rint(q) & 0xffu;
  const double a = fabs(q);
  const int e = a < 0x1p-6 ? -6 : ilogb(a);
  const double step = scalbn(1.0, e - 3);
  const float v = (float)copysign(rint(a / step) * step, q);  // an e4m3 value, or 480, which becomes 448
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xffu;
}
// Codes of x * mul / s for a re-quantised page, where two products would have to be compared: the quotient in 64 bits, whose error
// (2^-53) no quotient of such numbers is closer to a border than, unless it is a tie.  Not in line: it would take its callers'
// registers.
template <bool I8>
static __device__ __noinline__ uint32_t exact4(float x0, float x1, float x2, float x3, float mul, float s) {
  return code_of_double<I8>((double)x0 * (double)mul / (double)s) | (code_of_double<I8>((double)x1 * (double)mul / (double)s) << 8) |
         (code_of_double<I8>((double)x2 * (double)mul / (double)s) << 16) | (code_of_double<I8>((double)x3 * (double)mul / (double)s) << 24);
}
__device__ __forceinline__ uint32_t settled_i8(float q, float x, float s) {
  const float r = (q + kMagic) - kMagic, e = q - r;
  if (fabsf(e) <= 0.5f - 0x1p-15f) return (uint32_t)(int)r & 0xffu;
  const float border = r + copysignf(0.5f, e), d = fmaf(-border, s, x);
  const int low = (int)(border - 0.5f);
  return (uint32_t)(low + (d > 0.f || (d == 0.f && (low & 1)))) & 0xffu;
}
__device__ __forceinline__ uint32_t settled_e4m3(float q, float x, float s) {
  const uint32_t sign = (__float_as_uint(x) >> 24) & 0x80u, bits = __float_as_uint(fabsf(q));
  float border;
  uint32_t low;  // the code below it
  if (bits < 0x3c800000u) {
    const float k = floorf(fabsf(q) * 0x1p9f);
    border = (k + 0.5f) * 0x1p-9f;
    low = (uint32_t)(int)k;
  } else {
    border = __uint_as_float((bits & 0xfff00000u) | 0x80000u);
    low = (bits >> 20) - 960u;
  }
  const float d = fmaf(-border, s, fabsf(x));
  return min(low + (d > 0.f || (d == 0.f && (low & 1u))), 126u) | sign;
}
__device__ __forceinline__ bool e4m3_border(float q) {
  const uint32_t a = __float_as_uint(q) & 0x7fffffffu;
  if (a < 0x3c800000u)  // below 2^-6 the codes are multiples of 2^-9; zero is one of them
    return a != 0u && fabsf(fabsf(q) * 0x1p9f - floorf(fabsf(q) * 0x1p9f) - 0.5f) < 0x1p-18f;
  return ((a - 0x7fffcu) & 0xfffffu) <= 8u;
}
// codes of x / s (NEW: by = 1 / s rounded), or of x * mul / s (by = mul / s rounded)
template <bool I8, bool NEW>
__device__ __forceinline__ uint32_t nearest4(const float* x, float by, float mul, float s) {
  const float q[4] = {x[0] * by, x[1] * by, x[2] * by, x[3] * by};
  uint32_t r;
  bool open;
  if constexpr (I8) {
    float t[4], off = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = q[i] + kMagic;
      off = fmaxf(off, fabsf(q[i] - (t[i] - kMagic)));
    }
    r = __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040),
                    __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
    open = off > 0.5f - 0x1p-15f;
  } else {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(q[1]), "f"(q[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(q[3]), "f"(q[2]));
    r = (uint32_t)lo | ((uint32_t)hi << 16);
    open = e4m3_border(q[0]) | e4m3_border(q[1]) | e4m3_border(q[2]) | e4m3_border(q[3]);
  }
  if (open) {
    if constexpr (!NEW)
      r = exact4<I8>(x[0], x[1], x[2], x[3], mul, s);
    else if constexpr (I8)
      r = settled_i8(q[0], x[0], s) | (settled_i8(q[1], x[1], s) << 8) | (settled_i8(q[2], x[2], s) << 16) | (settled_i8(q[3], x[3], s) << 24);
    else
      r = settled_e4m3(q[0], x[0], s) | (settled_e4m3(q[1], x[1], s) << 8) | (settled_e4m3(q[2], x[2], s) << 16) | (settled_e4m3(q[3], x[3], s) << 24);
  }
  return r;
}

// ---- 16 bytes of a dense row ---------------------------------------------------------------------------------
template <typename T>
struct Chunk;  // floats of a 16-byte chunk, and the largest magnitude of many as bits that order like it
template <>
struct Chunk<float> {
  static __device__ __forceinline__ void floats(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint32_t top(uint32_t m, uint32_t w) { return max(m, w & 0x7fffffffu); }
  static __device__ __forceinline__ uint32_t top_bits(uint32_t m) { return m; }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Chunk<__nv_bfloat16> {
  static __device__ __forceinline__ void floats(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t top(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7fff7fffu); }
  static __device__ __forceinline__ uint32_t top_bits(uint32_t m) { return max(m >> 16, m & 0xffffu) << 16; }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Chunk<__half> {
  static __device__ __forceinline__ void floats(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint32_t top(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7fff7fffu); }
  static __device__ __forceinline__ uint32_t top_bits(uint32_t m) {
    const uint16_t h = (uint16_t)max(m >> 16, m & 0xffffu);
    return __float_as_uint(__half2float(*reinterpret_cast<const __half*>(&h)));
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7]));
  }
};
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load_chunk(const T* p) {
  if constexpr (VEC) {
    const float4 v = ldg_stream_f4(p);
    return make_uint4(__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w));
  }
  constexpr int E = 16 / sizeof(T);
  union {
    uint4 v;
    T e[E];
  } u;
#pragma unroll
  for (int i = 0; i < E; ++i) u.e[i] = p[i];
  return u.v;
}

template <bool I8>
__device__ __forceinline__ void codes_to_f32(uint32_t w, float (&f)[4]) {
  uint32_t a, b;
  codes_to_f16<I8>(w, a, b);
  const float2 x = __half22float2(*reinterpret_cast<__half2*>(&a)), y = __half22float2(*reinterpret_cast<__half2*>(&b));
  f[0] = x.x, f[1] = x.y, f[2] = y.x, f[3] = y.y;
}

// A warp's place: 16 slots of one (page, side, head).
struct IoTile {
  BlockPiece p;
  int side, head, part, page, tok0, page_tok0, start;  // part: which 16 slots of the page; page < 0: nothing to do
};
__device__ __forceinline__ IoTile io_tile(const BlocksIo& a, int64_t team, int part) {
  IoTile t;
  t.head = (int)(team % a.c.Hkv);
  const int64_t rest = team / a.c.Hkv;
  t.side = (int)(rest & 1);
  t.part = part;
  t.page = -1;
  t.page_tok0 = t.tok0 = t.start = 0;
  if ((rest >> 1) >= a.slots) return t;  // the whole team; find_piece() is for whole warps
  t.p = find_piece(a.c, a.r, (int)(rest >> 1), a.shift, 2);
  if (t.p.b < 0 || t.p.end < 0 || t.p.n == 0) return t;
  t.start = t.p.end - t.p.n;
  const int block = (t.start >> a.shift) + t.p.j;
  t.page_tok0 = block << a.shift;
  t.tok0 = t.page_tok0 + 16 * part;
  if (t.page_tok0 >= t.p.end) return t;
  t.page = a.c.block_table[(int64_t)t.p.b * a.c.max_blocks + block];
  if (t.page < 0 || t.page >= a.c.n_pages) {
    bad_status(a.c, SPHKV_ST_BAD_BLOCK);
    t.page = -2;
  }
  return t;
}

// A (page, side, head) belongs to page_size / 16 warps of one CTA; a warp holds its 16 rows as raw 16-byte chunks between the
// search for the largest magnitude and the rounding, so keys and values are read once.  Consecutive teams are heads of one
// page: their rows lie side by side in the dense tensors.
//
// Loads are made whether or not their row is wanted, from the nearest row that is (twice the same row leaves the largest magnitude as
// it is): a load that may be skipped ends in a copy that waits for it, and 16 of them one after the other are what a tile takes.
template <typename T, int DH, bool I8, bool VEC>
__global__ void __launch_bounds__(kIoThreads, sizeof(T) * DH == 512 ? 2 : 4) blocks_append_kernel(const BlocksIo a) {
  constexpr int E = 16 / sizeof(T), LPR = DH / E, RPL = 32 / LPR, L = 16 / RPL;  // lanes a row, rows a load, loads
  __shared__ uint32_t tops[kIoThreads / 32];
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = a.c.page_size >> 4;
  const IoTile t = io_tile(a, (int64_t)blockIdx.x * (kIoThreads / 32 / parts) + warp / parts, warp & (parts - 1));
  const bool live = t.page >= 0;
  const int64_t at = live ? (int64_t)t.page * a.c.Hkv + t.head : 0;
  float* const scale_at = (t.side ? a.c.v_scale : a.c.k_scale) + at;
  uint8_t* const codes = reinterpret_cast<uint8_t*>(t.side ? a.c.v_codes : a.c.k_codes) + ((at << a.shift) + 16 * t.part) * DH;
  const bool begun = live && t.start > t.page_tok0;
  const int first_new = t.start - t.tok0;                      // of this tile's rows, first_new .. end - 1 are new
  const int end = live ? min(16, t.p.end - t.tok0) : 0;
  const float s_old = begun ? *scale_at : 0.f;

  uint4 raw[L];
  uint32_t m = 0;
  const T* src = reinterpret_cast<const T*>(a.src[t.side]) + (int64_t)t.head * a.head_stride[t.side] + (lane % LPR) * E;
  const int lowest = max(first_new, 0);
  if (lowest < end) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int row = min(max(i * RPL + lane / LPR, lowest), end - 1);
      raw[i] = load_chunk<T, VEC>(src + (int64_t)(t.p.row0 + row - first_new) * a.row_stride[t.side]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < L; ++i) raw[i] = make_uint4(0, 0, 0, 0);
  }
  constexpr int OL = DH / 32, OLPR = DH / 16;  // held codes: 16 of a row per lane
  uint4 held[OL];
  const bool holds = begun && first_new > 0;
  if (holds) {
#pragma unroll
    for (int i = 0; i < OL; ++i) {
      const int row = min(i * (32 / OLPR) + lane / OLPR, first_new - 1);
      held[i] = *reinterpret_cast<const uint4*>(codes + row * DH + (lane % OLPR) * 16);
    }
  }
#pragma unroll
  for (int i = 0; i < L; ++i) {
    m = Chunk<T>::top(m, raw[i].x);
    m = Chunk<T>::top(m, raw[i].y);
    m = Chunk<T>::top(m, raw[i].z);
    m = Chunk<T>::top(m, raw[i].w);
  }
  // magnitudes order like their bits, infinities and NaN last
  m = __reduce_max_sync(0xffffffffu, Chunk<T>::top_bits(m));
  if (parts > 1) {
    if (lane == 0) tops[warp] = m;
    __syncthreads();
    for (int i = 0; i < parts; ++i) m = max(m, tops[(warp & ~(parts - 1)) + i]);
  }
  if (!live) return;
  float s = __uint_as_float(m);
  if (m < 0x7f800000u) {
    s = __fdiv_rn(s, I8 ? 127.f : 448.f);
    if (s < 0x1p-126f) s = 0.f;
  }
  bool grown = true;
  if (begun) {
    grown = __float_as_uint(s) > (__float_as_uint(s_old) & 0x7fffffffu);
    if (!grown) s = s_old;
  }
  if (t.part == 0 && lane == 0 && grown) *scale_at = s;  // parts > 1: all have read s_old before the barrier
  const bool finite = (__float_as_uint(s) & 0x7f800000u) != 0x7f800000u && s != 0.f;
  auto round_new = [&](auto lifted, float by, float inv) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int row = i * RPL + lane / LPR;
      if (row < first_new || row >= end) continue;
      uint32_t w[E / 4];
      float f[E];
      Chunk<T>::floats(raw[i], f);
      if constexpr (decltype(lifted)::value)
#pragma unroll
        for (int k = 0; k < E; ++k) f[k] *= kLift;
#pragma unroll
      for (int k = 0; k < E / 4; ++k) {
        w[k] = 0;
        if (finite) w[k] = nearest4<I8, true>(f + 4 * k, inv, 1.f, by);
      }
      uint8_t* to = codes + row * DH + (lane % LPR) * E;
      if constexpr (E == 8)
        *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
      else
        *reinterpret_cast<uint32_t*>(to) = w[0];
    }
  };
  if (s < kLeastScale)  // the whole warp: a branch of its own, since a product more per element is 2 % of the kernel
    round_new(std::true_type(), s * kLift, finite ? __frcp_rn(s * kLift) : 0.f);
  else
    round_new(std::false_type(), s, finite ? __frcp_rn(s) : 0.f);
  if (holds && grown) {
    const float ratio = finite ? __fdiv_rn(s_old, s) : 0.f;
#pragma unroll
    for (int i = 0; i < OL; ++i) {
      const int row = i * (32 / OLPR) + lane / OLPR;
      if (row >= first_new) continue;
      uint32_t w[4] = {held[i].x, held[i].y, held[i].z, held[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[4];
        codes_to_f32<I8>(w[k], f);
        w[k] = 0;
        if (finite) w[k] = nearest4<I8, false>(f, ratio, s_old, s);
      }
      *reinterpret_cast<uint4*>(codes + row * DH + (lane % OLPR) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// A lane takes as many codes at a time as make 16 bytes of output.
template <typename T, int DH, bool I8>
__global__ void __launch_bounds__(kIoThreads) blocks_read_kernel(const BlocksIo a) {
  constexpr int E = 16 / sizeof(T), LPR = DH / E, RPL = 32 / LPR, L = 16 / RPL;
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = a.c.page_size >> 4;
  const IoTile t = io_tile(a, (int64_t)blockIdx.x * (kIoThreads / 32 / parts) + warp / parts, warp & (parts - 1));
  if (t.page == -1) return;
  const bool live = t.page >= 0;
  const int64_t at = live ? (int64_t)t.page * a.c.Hkv + t.head : 0;
  const float s = live ? (t.side ? a.c.v_scale : a.c.k_scale)[at] : 0.f;
  const uint8_t* codes = reinterpret_cast<const uint8_t*>(t.side ? a.c.v_codes : a.c.k_codes) + ((at << a.shift) + 16 * t.part) * DH;
  const int first = t.start - t.tok0, end = min(16, t.p.end - t.tok0);
  uint32_t w[L][E / 4];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const uint8_t* from = codes + (i * RPL + lane / LPR) * DH + (lane % LPR) * E;  // all 16 rows are a page's, wanted or not
    if constexpr (E == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(from);
      w[i][0] = v.x, w[i][1] = v.y;
    } else {
      w[i][0] = *reinterpret_cast<const uint32_t*>(from);
    }
  }
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int row = i * RPL + lane / LPR;
    if (row < first || row >= end) continue;
    float f[E];
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      float g[4];
      codes_to_f32<I8>(w[i][k], g);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[4 * k + j] = live ? g[j] * s : 0.f;
    }
    T* to = reinterpret_cast<T*>(a.dst[t.side]) + ((int64_t)(t.p.row0 + row - first) * a.c.Hkv + t.head) * DH + (lane % LPR) * E;
    *reinterpret_cast<uint4*>(to) = Chunk<T>::pack(f);
  }
}

int check_blocks(const sphkv_blocks* c, const char* what) {
  SPHKV_REQUIRE(c != nullptr, SPHKV_E_ARG, "%s: cache is NULL", what);
  SPHKV_REQUIRE(c->k_codes && c->v_codes && c->k_scale && c->v_scale && c->block_table && c->ends, SPHKV_E_ARG,
                "%s: a required pointer is NULL", what);
  SPHKV_REQUIRE(c->dh == 64 || c->dh == 128, SPHKV_E_ARG, "%s: dh=%d (64 or 128)", what, c->dh);
  SPHKV_REQUIRE(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128, SPHKV_E_ARG,
                "%s: page_size=%d (16, 32, 64 or 128)", what, c->page_size);
  SPHKV_REQUIRE(c->B > 0 && c->Hkv > 0 && c->n_pages > 0 && c->max_blocks > 0, SPHKV_E_ARG, "%s: B=%d Hkv=%d n_pages=%d max_blocks=%d",
                what, c->B, c->Hkv, c->n_pages, c->max_blocks);
  SPHKV_REQUIRE(c->store == SPHKV_BLOCKS_I8 || c->store == SPHKV_BLOCKS_E4M3, SPHKV_E_DTYPE, "%s: store=%d", what, c->store);
  SPHKV_REQUIRE((((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15) == 0, SPHKV_E_ALIGN, "%s: codes need 16 B", what);
  // rows of the pools are numbered in 32 bits, and so are a sequence's tokens
  SPHKV_REQUIRE((int64_t)c->n_pages * c->Hkv * c->page_size <= 0x7fffffff, SPHKV_E_LIMIT, "%s: %lld rows of pages (max 2^31 - 1)", what,
                (long long)c->n_pages * c->Hkv * c->page_size);
  SPHKV_REQUIRE((int64_t)c->max_blocks * c->page_size <= 0x40000000 && c->B <= 0x100000, SPHKV_E_LIMIT,
                "%s: max_blocks * page_size above 2^30, or B above 2^20", what);
  return 0;
}

int block_rows(BlockRows& r, const sphkv_blocks* c, const int32_t* cu, int64_t rows, const char* what) {
  SPHKV_REQUIRE(rows >= 0 && rows <= 0x1fffffff, SPHKV_E_LIMIT, "%s: rows=%lld (0 .. 2^29 - 1)", what, (long long)rows);
  SPHKV_REQUIRE(cu != nullptr || rows % c->B == 0, SPHKV_E_ARG, "%s: %lld rows are not the same number for each of %d sequences", what,
                (long long)rows, c->B);
  r.cu = cu;
  r.rows = (int)rows;
  r.even = (int)(rows / c->B);
  r.mul = 1;
  r.lone = false;
  return 0;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int make_codes_map(CUtensorMap* map, const sphkv_blocks& c, void* codes, int box_rows, const char* what) {
  static const EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult found;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) == cudaSuccess &&
                    found == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeTiledFn>(ptr) : nullptr;
  }();
  SPHKV_REQUIRE(fn != nullptr, SPHKV_E_ARG, "%s: cuTensorMapEncodeTiled is not available from this driver", what);
  const cuuint64_t dims[2] = {(cuuint64_t)c.dh, (cuuint64_t)c.n_pages * c.Hkv * c.page_size};
  const cuuint64_t strides[1] = {(cuuint64_t)c.dh};
  const cuuint32_t box[2] = {(cuuint32_t)c.dh, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult rc = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         c.dh == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  SPHKV_REQUIRE(rc == CUDA_SUCCESS, SPHKV_E_ARG, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)rc);
  return 0;
}

static int log2_of(int n) { return n == 16 ? 4 : n == 32 ? 5 : n == 64 ? 6 : 7; }

static int64_t io_blocks(BlocksIo& a) {
  a.shift = log2_of(a.c.page_size);
  const int64_t slots = block_slots(a.r, a.c.B, a.shift, 2);
  a.slots = (int)slots;
  const int64_t per = kIoThreads / 32 / (a.c.page_size / 16);
  return (slots * 2 * a.c.Hkv + per - 1) / per;
}

template <typename T, int DH, bool READ>
static int launch_io(const BlocksIo& a, int64_t blocks, cudaStream_t st) {
  if constexpr (READ) {
    auto k = a.c.store == SPHKV_BLOCKS_I8 ? blocks_read_kernel<T, DH, true> : blocks_read_kernel<T, DH, false>;
    (void)launch_overlapped(k, dim3((unsigned)blocks), dim3(kIoThreads), 0, st, a);
    return check_launch("blocks_read_kernel");
  } else {
    auto k = a.c.store == SPHKV_BLOCKS_I8 ? (a.vec ? blocks_append_kernel<T, DH, true, true> : blocks_append_kernel<T, DH, true, false>)
                                          : (a.vec ? blocks_append_kernel<T, DH, false, true> : blocks_append_kernel<T, DH, false, false>);
    (void)launch_overlapped(k, dim3((unsigned)blocks), dim3(kIoThreads), 0, st, a);
    return check_launch("blocks_append_kernel");
  }
}
template <bool READ>
static int launch_io_types(BlocksIo& a, int dtype, const char* what, cudaStream_t st) {
  const int64_t blocks = io_blocks(a);
  SPHKV_REQUIRE(blocks <= 0x7fffffff, SPHKV_E_LIMIT, "%s: too many pages for one launch", what);
  if (blocks == 0) return 0;
  if (a.c.dh == 128)
    return dtype == SPHKV_F32    ? launch_io<float, 128, READ>(a, blocks, st)
           : dtype == SPHKV_BF16 ? launch_io<__nv_bfloat16, 128, READ>(a, blocks, st)
                                 : launch_io<__half, 128, READ>(a, blocks, st);
  return dtype == SPHKV_F32    ? launch_io<float, 64, READ>(a, blocks, st)
         : dtype == SPHKV_BF16 ? launch_io<__nv_bfloat16, 64, READ>(a, blocks, st)
                               : launch_io<__half, 64, READ>(a, blocks, st);
}

}  // namespace sphkv

using namespace sphkv;

extern "C" int sphkv_blocks_append(const sphkv_blocks* c, const void* k, const void* v, int32_t dtype, int64_t k_row_stride,
                                   int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride, const int32_t* cu,
                                   int64_t rows, void* stream) {
  if (int rc = check_blocks(c, "blocks_append")) return rc;
  SPHKV_REQUIRE(dtype >= 0 && dtype <= 2, SPHKV_E_DTYPE, "blocks_append: dtype=%d", dtype);
  BlocksIo a = {};
  a.c = *c;
  if (int rc = block_rows(a.r, c, cu, rows, "blocks_append")) return rc;
  if (rows == 0) return 0;
  SPHKV_REQUIRE(k && v, SPHKV_E_ARG, "blocks_append: k or v is NULL");
  const int64_t size = dtype == SPHKV_F32 ? 4 : 2;
  SPHKV_REQUIRE((((uintptr_t)k | (uintptr_t)v) & (size - 1)) == 0, SPHKV_E_ALIGN, "blocks_append: k or v is not on an element's boundary");
  a.src[0] = k, a.src[1] = v;
  a.row_stride[0] = k_row_stride, a.row_stride[1] = v_row_stride;
  a.head_stride[0] = k_head_stride, a.head_stride[1] = v_head_stride;
  a.vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 &&
          (((k_row_stride | k_head_stride | v_row_stride | v_head_stride) * size) & 15) == 0;
  return launch_io_types<false>(a, dtype, "blocks_append", reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int sphkv_blocks_read(const sphkv_blocks* c, void* k_out, void* v_out, int32_t dtype, const int32_t* cu, int64_t rows,
                                 void* stream) {
  if (int rc = check_blocks(c, "blocks_read")) return rc;
  SPHKV_REQUIRE(dtype >= 0 && dtype <= 2, SPHKV_E_DTYPE, "blocks_read: dtype=%d", dtype);
  BlocksIo a = {};
  a.c = *c;
  if (int rc = block_rows(a.r, c, cu, rows, "blocks_read")) return rc;
  if (rows == 0) return 0;
  SPHKV_REQUIRE(k_out && v_out, SPHKV_E_ARG, "blocks_read: k_out or v_out is NULL");
  SPHKV_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, SPHKV_E_ALIGN, "blocks_read: outputs need 16 B");
  a.dst[0] = k_out, a.dst[1] = v_out;
  return launch_io_types<true>(a, dtype, "blocks_read", reinterpret_cast<cudaStream_t>(stream));
}
