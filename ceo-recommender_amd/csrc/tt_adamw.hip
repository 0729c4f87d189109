// AdamW over a list of tensors (gfx950), states in 32 or in 8 bits.
//
//   m' = m + (1 - b1)(g - m);  v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// k_adamw takes up to ADAMW_LIST tensors by value (kernel arguments, so a
// captured graph keeps them): a workgroup finds its tensor from the prefix of
// chunk counts, then walks its chunk 8 consecutive values a thread.
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
  float w1, b2, c2, eps, decay;
  float *m, *v;
  uint8_t *mc, *ms, *rc, *rs;
  int64_t* steps;
  AdamwCoef* coefs;
  double lr, b1d, b2d;
  uint64_t seed;
};
static_assert(sizeof(AdamwArgs) <= 4096, "kernel arguments");

// device step counters: one thread a tensor, before k_adamw
__global__ __launch_bounds__(ADAMW_LIST) void k_adamw_advance(AdamwArgs a) {
  const int k = (int)threadIdx.x;
  if (k >= a.n_t) return;
  const uint32_t i = a.c[k].key_lo;
  const int64_t t = ++a.steps[i];
  a.coefs[i] = adamw_coef(a.lr, a.b1d, a.b2d, a.seed, t);
}

struct AdamwHp {
  float w1, b2, c2, eps, decay;
};

// p, m, v in; p', m', v' out; returns sqrt(v')
__device__ __forceinline__ float adamw_elem(float& p, float& m, float& v, float g, const AdamwHp& h,
                                            const AdamwCoef& c) {
  m = m + h.w1 * (g - m);
  v = v * h.b2 + (h.c2 * g) * g;
  const float r = sqrtf(v);
  p = p * h.decay - c.step_size * (m / (r / c.bc2s + h.eps));
  return r;
}

template <int BITS, int DT>
__device__ __forceinline__ void adamw_chunk(const AdamwArgs& a, int k, const AdamwCoef& c, int64_t from) {
  using namespace b8;
  const AdamwHp h{a.w1, a.b2, a.c2, a.eps, a.decay};
  void* const P = a.p[k];
  const void* const G = a.g[k];
  const int64_t n = a.n[k], blk0 = a.blk[k];
  const int64_t to = min(from + (int64_t)a.chunk, n);
  for (int64_t i = from + (int64_t)threadIdx.x * 8; i - (int64_t)(threadIdx.x % LANES) * 8 < to; i += ADAMW_STRIDE) {
    // the 16 lanes of a block stay together; lanes past the tensor's end see zeros
    const int live = (int)max((int64_t)0, min((int64_t)8, n - i));
    const int64_t s = blk0 * BLK + i;
    float p[8], g[8], m[8], v[8];
    ld8n<DT>(P, i, live, p);
    ld8n<DT>(G, i, live, g);
    if constexpr (BITS == 32) {
      ld8<TT_F32>(a.m, s, m);
      ld8<TT_F32>(a.v, s, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) adamw_elem(p[e], m[e], v[e], g[e], h, c);
      if (live < 8)  // the padding stays zero
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e >= live) m[e] = v[e] = 0.f;
      st8<TT_F32>(a.m, s, m);
      st8<TT_F32>(a.v, s, v);
    } else {
      const int64_t b = blk0 + (i / BLK);
      u32x2 mc, rc;
      __builtin_memcpy(&mc, a.mc + s, 8);
      __builtin_memcpy(&rc, a.rc + s, 8);
      const float sm = scale_of(a.ms[b]), sr = scale_of(a.rs[b]);
      float r[8];
      uint32_t am = 0, ar = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t cm = (mc[e / 4] >> (8 * (e % 4))) & 0xFFu, cr = (rc[e / 4] >> (8 * (e % 4))) & 0xFFu;
        const float nan = __uint_as_float(0x7FC00000u);
        const float mag = (cm & 0x7Fu) == NAN_M ? nan : code_value<MANT_M>(cm & 0x7Fu, sm);
        m[e] = (cm & 0x80u) ? -mag : mag;
        const float root = cr == NAN_R ? nan : code_value<MANT_R>(cr, sr);
        v[e] = root * root;
        r[e] = adamw_elem(p[e], m[e], v[e], g[e], h, c);
        const uint32_t bm = __float_as_uint(m[e]) & 0x7FFFFFFFu, br = __float_as_uint(r[e]);
        am = max(am, finite_bits(bm) ? bm : 0u);
        ar = max(ar, finite_bits(br) ? br : 0u);  // a NaN's sign bit, too, is over the finite ones
      }
      const uint32_t ym = (uint32_t)scale_byte(row_max16(am), CARRY_M);
      const uint32_t yr = (uint32_t)scale_byte(row_max16(ar), CARRY_R);
      const float im = inv_scale(ym), ir = inv_scale(yr);
      const uint32_t rk = perm32((uint32_t)b ^ c.key_lo) + c.key_hi;
      mc = rc = (u32x2){0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t u = perm32(rk ^ ((uint32_t)((i % BLK) + e) * 0x9E3779B9u));
        const uint32_t bm = __float_as_uint(m[e]);
        uint32_t cm = finite_bits(bm & 0x7FFFFFFFu) ? round_code<MANT_M>(fabsf(m[e]) * im, u & 0xFFFFu) : NAN_M;
        cm |= (bm >> 24) & 0x80u;
        uint32_t cr = finite_bits(__float_as_uint(r[e])) ? round_code<MANT_R>(r[e] * ir, u >> 16) : NAN_R;
        cr = r[e] > 0.f ? max(cr, 1u) : cr;  // a positive root stays positive: m' / sqrt(v') stays bounded
        mc[e / 4] |= cm << (8 * (e % 4));
        rc[e / 4] |= cr << (8 * (e % 4));
      }
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
  const AdamwCoef c = a.steps ? a.coefs[a.c[k].key_lo] : a.c[k];
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
    const float s = scale_of(scales[i / LANES]);
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
