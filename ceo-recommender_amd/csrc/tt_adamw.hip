// AdamW over a list of tensors (gfx950), states in 32 or in 8 bits.
//
//   m' = m + (1 - b1)(g - m), for b1 < 1/2 g - b1 (g - m): the rounding of g - m
//   by the smaller factor;  v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// k_adamw takes up to ADAMW_LIST tensors by value (kernel arguments, so a
// captured graph keeps them): a workgroup finds its tensor from the prefix of
// chunk counts, one lane a tensor, then walks its chunk.
//
// 32-bit states are bound by memory (28 bytes a value in fp32): 96 M values
// 498 us, 5.4 TB/s; in bf16 402 us.  8-bit states in bf16 (10 bytes a value) by
// instructions, about 60 a value of which the rounding hash takes 15: 96 M values
// 215-240 us, fp16 224, fp32 302 us (5.1 TB/s); reading the values back
// (k_adamw_held) 95 us, 6.1 TB/s.  The 21 tensors of the two towers take 3.6 and
// 4.4 us, launch and latency.
#include "tt_block8.h"

namespace tt {

constexpr int ADAMW_LIST = 64;     // tensors per launch: one lane each finds a workgroup's tensor
constexpr int ADAMW_THREADS = 256;
constexpr int ADAMW_STRIDE = ADAMW_THREADS * 8;  // values a workgroup covers at once: 16 blocks

struct AdamwCoef {  // what depends on t
  float step_size, bc2s;
  uint32_t key_lo, key_hi;  // of the rounding hash
};

__host__ __device__ __forceinline__ AdamwCoef adamw_coef(double lr, double b1, double b2, uint64_t seed, int64_t t) {
  AdamwCoef c;
  c.step_size = (float)(lr / (1.0 - pow(b1, (double)t)));
  c.bc2s = (float)sqrt(1.0 - pow(b2, (double)t));
  const uint64_t key = mix64(seed * 0x9E3779B97F4A7C15ull + (uint64_t)t * 0xD1B54A32D192ED03ull);
  c.key_lo = (uint32_t)key;
  c.key_hi = (uint32_t)(key >> 32);
  return c;
}

struct AdamwArgs {
  void* p[ADAMW_LIST];
  const void* g[ADAMW_LIST];
  int64_t n[ADAMW_LIST], blk[ADAMW_LIST];
  AdamwCoef c[ADAMW_LIST];     // host steps; key_lo holds the counter's index with device steps
  uint8_t dtype[ADAMW_LIST];
  int32_t first[ADAMW_LIST];   // first chunk of the tensor; INT32_MAX past the list
  int32_t chunk;               // values per chunk, a multiple of ADAMW_STRIDE
  int32_t n_t;
  float w1, b2, c2, eps, decay;  // w1: 1 - b1, or -b1 with from_grad
  int32_t from_grad;
  float *m, *v;
  uint8_t *mc, *ms, *rc, *rs;
  const AdamwCoef* coefs;      // device steps, or null
};
static_assert(sizeof(AdamwArgs) <= 4096, "kernel arguments");

// device step counters: one thread a counter, each named once, before any k_adamw of the call
struct AdamwCounters {
  int64_t* steps;
  AdamwCoef* coefs;
  double lr, b1, b2;
  uint64_t seed;
  uint32_t at[ADAMW_LIST];
  int32_t n;
};
__global__ __launch_bounds__(ADAMW_LIST) void k_adamw_advance(AdamwCounters a) {
  const int k = (int)threadIdx.x;
  if (k >= a.n) return;
  const uint32_t i = a.at[k];
  const int64_t t = ++a.steps[i];
  a.coefs[i] = adamw_coef(a.lr, a.b1, a.b2, a.seed, t);
}

struct AdamwHp {
  float w1, b2, c2, eps, decay;
  bool from_grad;
};

__device__ __forceinline__ void adamw_moments(float& m, float& v, float g, const AdamwHp& h) {
  m = (h.from_grad ? g : m) + h.w1 * (g - m);
  v = v * h.b2 + (h.c2 * g) * g;
}
// 32-bit states: correctly rounded root and quotients
__device__ __forceinline__ void adamw_elem(float& p, float& m, float& v, float g, const AdamwHp& h, const AdamwCoef& c) {
  adamw_moments(m, v, g, h);
  p = p * h.decay - c.step_size * (m / (sqrtf(v) / c.bc2s + h.eps));
}

// Roots of a thread's 8 values of v' (8-bit states, whose kernel the
// instructions bound): the hardware's square root, off by one unit in the last
// place, for the correctly rounded one of about 12 instructions; the same for
// the reciprocal in the update.  The hardware takes subnormal input as zero, so
// a wave that holds such values takes their roots of v' 2^64.
__device__ __forceinline__ void roots8(const float (&v)[8], float (&r)[8]) {
  uint32_t least = ~0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    r[e] = __builtin_amdgcn_sqrtf(v[e]);
    least = min(least, __float_as_uint(v[e]));
  }
  if (__ballot(least < 0x00800000u)) {
    asm volatile("");  // a branch: zeros are common, subnormals are not
    least = ~0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) least = min(least, __float_as_uint(v[e]) - 1u);  // zero goes to the top
    if (__ballot(least < 0x007FFFFFu)) {
      asm volatile("");
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (__float_as_uint(v[e]) < 0x00800000u) r[e] = __builtin_amdgcn_sqrtf(v[e] * 0x1p64f) * 0x1p-32f;
    }
  }
}

// whether a byte of w is 0xFF (and at times where one is 0xFE below a 0xFF: never without one)
__device__ __forceinline__ bool has_ff(uint32_t w) { return ((~w - 0x01010101u) & w & 0x80808080u) != 0; }

template <int BITS, int DT>
__device__ __forceinline__ void adamw_chunk(const AdamwArgs& a, int k, const AdamwCoef& c, int64_t from) {
  using namespace b8;
  const AdamwHp h{a.w1, a.b2, a.c2, a.eps, a.decay, a.from_grad != 0};
  void* const P = a.p[k];
  const void* const G = a.g[k];
  const int64_t n = a.n[k], blk0 = a.blk[k];
  const int64_t to = min(from + (int64_t)a.chunk, n);
  const float inv_bc2s = 1.f / c.bc2s;
  if constexpr (BITS == 32) {
    // 4 values a thread, twice: every access of a wave covers whole lines
    constexpr int PER = 4, HALF = ADAMW_STRIDE / 2;
    int64_t at = from;
    for (; at + ADAMW_STRIDE <= to; at += ADAMW_STRIDE) {  // no tests between the loads
      const int64_t i = at + (int64_t)threadIdx.x * PER;
      float p[2][PER], g[2][PER], m[2][PER], v[2][PER];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        ldv<DT, PER>(P, i + q * HALF, p[q]);
        ldv<DT, PER>(G, i + q * HALF, g[q]);
        ldv<TT_F32, PER>(a.m, blk0 * BLK + i + q * HALF, m[q]);
        ldv<TT_F32, PER>(a.v, blk0 * BLK + i + q * HALF, v[q]);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int e = 0; e < PER; ++e) adamw_elem(p[q][e], m[q][e], v[q][e], g[q][e], h, c);
        stv<DT, PER>(P, i + q * HALF, p[q]);
        stv<TT_F32, PER>(a.m, blk0 * BLK + i + q * HALF, m[q]);
        stv<TT_F32, PER>(a.v, blk0 * BLK + i + q * HALF, v[q]);
      }
    }
    for (int64_t i = at + (int64_t)threadIdx.x * PER; i < to; i += HALF) {
      const int live = (int)min((int64_t)PER, to - i);
      float p[PER], g[PER], m[PER], v[PER];
      ldn<DT, PER>(P, i, live, p);
      ldn<DT, PER>(G, i, live, g);
      ldn<TT_F32, PER>(a.m, blk0 * BLK + i, live, m);
      ldn<TT_F32, PER>(a.v, blk0 * BLK + i, live, v);
#pragma unroll
      for (int e = 0; e < PER; ++e) adamw_elem(p[e], m[e], v[e], g[e], h, c);
      stn<DT, PER>(P, i, live, p);
      stn<TT_F32, PER>(a.m, blk0 * BLK + i, live, m);  // (the padding stays zero)
      stn<TT_F32, PER>(a.v, blk0 * BLK + i, live, v);
    }
    return;
  }
  uint32_t place[8];  // of the hash: this thread's values keep their places in their blocks
#pragma unroll
  for (int e = 0; e < 8; ++e) place[e] = (threadIdx.x % LANES * 8 + e) * 0x9E3779B9u;
  for (int64_t i = from + (int64_t)threadIdx.x * 8; i - (int64_t)(threadIdx.x % LANES) * 8 < to; i += ADAMW_STRIDE) {
    // the 16 lanes of a block stay together; lanes past the tensor's end see zeros
    const int live = (int)max((int64_t)0, min((int64_t)8, n - i));
    const int64_t s = blk0 * BLK + i;
    float p[8], g[8], m[8], v[8];
    ld8n<DT>(P, i, live, p);
    ld8n<DT>(G, i, live, g);
    {
      const int64_t b = blk0 + (i / BLK);
      u32x2 mc, rc;
      __builtin_memcpy(&mc, a.mc + s, 8);
      __builtin_memcpy(&rc, a.rc + s, 8);
      const uint32_t bm = a.ms[b], br = a.rs[b];
      decode8(mc, scale_of(bm), m);  // e4m3: the hardware's conversion, NaN and signs with it
      float r[8], root[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) root[e] = code_value<MANT_R>((rc[e / 4] >> (8 * (e % 4))) & 0xFFu, br);
      if (__ballot(has_ff(rc[0]) || has_ff(rc[1]))) {
        asm volatile("");
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (((rc[e / 4] >> (8 * (e % 4))) & 0xFFu) == NAN_R) root[e] = __uint_as_float(0x7FC00000u);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = root[e] * root[e];
        adamw_moments(m[e], v[e], g[e], h);
      }
      roots8(v, r);
      uint32_t am = 0, ar = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = p[e] * h.decay - c.step_size * (m[e] * __builtin_amdgcn_rcpf(r[e] * inv_bc2s + h.eps));
        am = max(am, __float_as_uint(m[e]) & 0x7FFFFFFFu);
        ar = max(ar, __float_as_uint(r[e]));  // a root's sign bit is a NaN's
      }
      const bool odd = !finite_bits(am) || !finite_bits(ar);
      u32x2 nan_m = {0u, 0u}, nan_r = {0u, 0u};
      if (__ballot(odd)) {  // infinities or NaN somewhere in the wave: held as NaN, the others by the finite ones
        asm volatile("");    // a branch, not 40 selects
        am = ar = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t xm = __float_as_uint(m[e]) & 0x7FFFFFFFu, xr = __float_as_uint(r[e]);
          if (!finite_bits(xm)) m[e] = 0.f, nan_m[e / 4] |= NAN_M << (8 * (e % 4));
          if (!finite_bits(xr)) r[e] = 0.f, nan_r[e / 4] |= NAN_R << (8 * (e % 4));
          am = max(am, finite_bits(xm) ? xm : 0u);
          ar = max(ar, finite_bits(xr) ? xr : 0u);
        }
      }
      const uint32_t ym = (uint32_t)scale_byte(row_max16(am), CARRY_M);
      const uint32_t yr = (uint32_t)scale_byte(row_max16(ar), CARRY_R);
      const uint32_t rk = perm32((uint32_t)b ^ c.key_lo) + c.key_hi;
      mc = rc = (u32x2){0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t u = perm32(rk ^ place[e]);
        const uint32_t xm = __float_as_uint(m[e]), xr = __float_as_uint(r[e]);
        const uint32_t cm = round_code<MANT_M>(fabsf(m[e]), ym, u & 0xFFFFu) | (xm >> 24 & 0x80u);
        // a positive root stays positive: m' / sqrt(v') stays bounded
        const uint32_t cr = max(round_code<MANT_R>(r[e], yr, u >> 16), min(xr, 1u));
        mc[e / 4] |= cm << (8 * (e % 4));
        rc[e / 4] |= cr << (8 * (e % 4));
      }
      mc |= nan_m;
      rc |= nan_r;
      if (live < 8) {  // the padding stays zero
        const uint64_t keep = live > 0 ? ~0ull >> (64 - 8 * live) : 0ull;
        mc[0] &= (uint32_t)keep, mc[1] &= (uint32_t)(keep >> 32);
        rc[0] &= (uint32_t)keep, rc[1] &= (uint32_t)(keep >> 32);
      }
      __builtin_memcpy(a.mc + s, &mc, 8);
      __builtin_memcpy(a.rc + s, &rc, 8);
      if (threadIdx.x % LANES == 0) {
        a.ms[b] = (uint8_t)ym;
        a.rs[b] = (uint8_t)yr;
      }
    }
    st8n<DT>(P, i, live, p);
  }
}

template <int BITS>
__global__ __launch_bounds__(ADAMW_THREADS) void k_adamw(AdamwArgs a) {
  // this workgroup's tensor: the last whose first chunk is not after it
  const uint64_t le = __ballot(a.first[lane_id()] <= (int32_t)blockIdx.x);
  const int k = __builtin_amdgcn_readfirstlane(__popcll(le) - 1);
  const int64_t from = (int64_t)((int32_t)blockIdx.x - a.first[k]) * a.chunk;
  const AdamwCoef c = a.coefs ? a.coefs[a.c[k].key_lo] : a.c[k];
  switch (a.dtype[k]) {
    case TT_F32: adamw_chunk<BITS, TT_F32>(a, k, c, from); break;
    case TT_BF16: adamw_chunk<BITS, TT_BF16>(a, k, c, from); break;
    default: adamw_chunk<BITS, TT_F16>(a, k, c, from); break;
  }
}

// the values that 8-bit states stand for, in bfloat16 (exact): blockIdx.y = 0: m, 1: sqrt(v)
__global__ __launch_bounds__(256) void k_adamw_held(const uint8_t* mc, const uint8_t* ms, const uint8_t* rc,
                                                    const uint8_t* rs, void* m, void* r, int64_t n8) {
  using namespace b8;
  const bool root = blockIdx.y != 0;
  const uint8_t* codes = root ? rc : mc;
  const uint8_t* scales = root ? rs : ms;
  void* out = root ? r : m;
  const float nan = __uint_as_float(0x7FC00000u);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += (int64_t)gridDim.x * blockDim.x) {
    u32x2 w;
    __builtin_memcpy(&w, codes + i * 8, 8);
    const uint32_t s = scales[i / LANES];
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t c = (w[e / 4] >> (8 * (e % 4))) & 0xFFu;
      const uint32_t mag = root ? c : c & 0x7Fu;
      const float y = root ? code_value<MANT_R>(mag, s) : code_value<MANT_M>(mag, s);
      const float z = mag == (root ? NAN_R : NAN_M) ? nan : y;
      x[e] = !root && (c & 0x80u) ? -z : z;
    }
    st8<TT_BF16>(out, i * 8, x);
  }
}

}  // namespace tt
