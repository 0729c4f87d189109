// The embedding catalogue in e4m3 blocks of 128 (gfx950): rows written and
// read back, queries scored against it, and the queries' gradient.
#include "tt_block8.h"

namespace tt {

struct CatRows {        // which catalogue row a call's row i is
  const int64_t* rows;  // nullable
  int64_t row0, capacity;
};
__device__ __forceinline__ int64_t cat_row(const CatRows& r, int64_t i) { return r.rows ? r.rows[i] : r.row0 + i; }
__device__ __forceinline__ bool cat_row_ok(const CatRows& r, int64_t c) { return c >= 0 && c < r.capacity; }

// A row named twice takes its last mention: every mention raises the row's
// owner to its own place + 1 (k_cat_own), then only the owner writes and puts
// the word back to zero (k_cat_write); a mention that lost sees either the
// owner's place or zero, never its own.
__global__ __launch_bounds__(256) void k_cat_own(CatRows r, int64_t m, int32_t* owner) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < m; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t c = r.rows[i];
    if (cat_row_ok(r, c)) atomicMax(owner + c, (int32_t)i + 1);
  }
}

// 16 lanes a block of 128: 8 values each
template <int DT>
__global__ __launch_bounds__(256) void k_cat_write(const void* x, int64_t m, int64_t ldx, int d, int nkb, CatRows r,
                                                   uint8_t* codes, uint8_t* scales, int32_t* owner) {
  using namespace b8;
  const int64_t total = m * nkb;
  for (int64_t u = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LANES; u < total;
       u += (int64_t)gridDim.x * blockDim.x / LANES) {
    const int64_t i = u / nkb;
    const int kb = (int)(u - i * nkb);
    const int64_t c = cat_row(r, i);
    if (!cat_row_ok(r, c)) continue;
    if (owner && owner[c] != (int32_t)i + 1) continue;
    const int k = kb * BLK + (int)(threadIdx.x % LANES) * 8;
    float v[8];
    ld8n<DT>(x, i * ldx + k, max(0, min(8, d - k)), v);
    uint32_t byte;
    const u32x2 w = encode8(v, byte);
    __builtin_memcpy(codes + (c * nkb + kb) * BLK + (threadIdx.x % LANES) * 8, &w, 8);
    if (threadIdx.x % LANES == 0) scales[c * nkb + kb] = (uint8_t)byte;
  }
}
__global__ __launch_bounds__(256) void k_cat_disown(CatRows r, int64_t m, int32_t* owner) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < m; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t c = r.rows[i];
    if (cat_row_ok(r, c)) owner[c] = 0;
  }
}

template <int DT>
__global__ __launch_bounds__(256) void k_cat_read(const uint8_t* codes, const uint8_t* scales, CatRows r, int64_t m,
                                                  int d, int nkb, void* out, int64_t ldo) {
  using namespace b8;
  const int64_t total = m * nkb;
  for (int64_t u = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LANES; u < total;
       u += (int64_t)gridDim.x * blockDim.x / LANES) {
    const int64_t i = u / nkb;
    const int kb = (int)(u - i * nkb);
    const int64_t c = cat_row(r, i);
    const int k = kb * BLK + (int)(threadIdx.x % LANES) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (cat_row_ok(r, c)) {
      u32x2 w;
      __builtin_memcpy(&w, codes + (c * nkb + kb) * BLK + (threadIdx.x % LANES) * 8, 8);
      decode8(w, scale_of(scales[c * nkb + kb]), v);
    }
    st8n<DT>(out, i * ldo + k, max(0, min(8, d - k)), v);
  }
}

// ---------------------------------------------------------------------------
// scores = Q^ C^^T.  Lane l supplies 32 bytes of operand row l & 15 for a block
// of 128 (which 32 is the same for both operands, so any order of k is right);
// C: lane l holds C[row = 4 (l >> 4) + reg][column = l & 15].
//
// Results in 16 bits: v_mfma_scale_f32_16x16x128_f8f6f4, one instruction a
// block, which takes both blocks' scale bytes, so the sums over all blocks
// stay in the accumulator.  The 8-bit matrix instructions cut the products of
// one instruction off below the largest of them (measured over all e4m3
// values: a sum of 128 is off by up to 2^-11 of its largest product, 5e-5 of
// the result in the 2-norm), far below the results' own rounding (2^-9, 2^-12)
// but not a sum in 32 bits.
// Results in 32 bits: both operands decoded to bf16, exactly, and
// v_mfma_f32_16x16x32_bf16, whose sums measured 8e-8.
// ---------------------------------------------------------------------------
typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma_block8(const i32x8& a, const i32x8& b, const f32x4& c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}
// 8 codes and their block's scale -> bf16, exact
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t lo, uint32_t hi, float s) {
  float x[8];
  b8::decode8((u32x2){lo, hi}, s, x);
  u32x4 w;
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = pk_bf16(x[2 * k], x[2 * k + 1]);
  return __builtin_bit_cast(bf16x8, w);
}
__device__ __forceinline__ f32x4 mfma_block_bf16(const i32x8& a, const i32x8& b, f32x4 c, int sa, int sb) {
  const float fa = b8::scale_of((uint32_t)sa), fb = b8::scale_of((uint32_t)sb);
#pragma unroll
  for (int h = 0; h < 4; ++h)
    c = mfma_bf16(codes_to_bf16((uint32_t)a[2 * h], (uint32_t)a[2 * h + 1], fa),
                  codes_to_bf16((uint32_t)b[2 * h], (uint32_t)b[2 * h + 1], fb), c);
  return c;
}

template <int DT>
__global__ __launch_bounds__(256) void k_cat_scores(const uint8_t* q, const uint8_t* qs, int64_t m,
                                                    const uint8_t* codes, const uint8_t* scales, int64_t n, int nkb,
                                                    void* out, int64_t n_tiles) {
  using namespace b8;
  const int l = lane_id(), w = wave_id();
  const int64_t tm = (int64_t)blockIdx.x / n_tiles, tn = (int64_t)blockIdx.x % n_tiles;
  const int64_t m0 = tm * 64 + (w >> 1) * 32, n0 = tn * 64 + (w & 1) * 32;
  f32x4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = zero4();
  int64_t rc[2], rq[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    rc[i] = min(n0 + 16 * i + (l & 15), n - 1);
    rq[i] = min(m0 + 16 * i + (l & 15), m - 1);
  }
  for (int kb = 0; kb < nkb; ++kb) {
    i32x8 a[2], b[2];
    int sa[2], sb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      __builtin_memcpy(&a[i], codes + (rc[i] * nkb + kb) * BLK + (l >> 4) * 32, 32);
      __builtin_memcpy(&b[i], q + (rq[i] * nkb + kb) * BLK + (l >> 4) * 32, 32);
      sa[i] = scales[rc[i] * nkb + kb];
      sb[i] = qs[rq[i] * nkb + kb];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        acc[i][j] = DT == TT_F32 ? mfma_block_bf16(a[i], b[j], acc[i][j], sa[i], sb[j])
                                 : mfma_block8(a[i], b[j], acc[i][j], sa[i], sb[j]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t row = m0 + 16 * j + (l & 15), col = n0 + 16 * i + 4 * (l >> 4) + e;
        if (row < m && col < n) st1<DT>(out, row * n + col, acc[i][j][e]);
      }
}

// ---------------------------------------------------------------------------
// dq = dS C^: C^ is exact in bf16, dS is split into bf16 planes that hold it
// exactly (bf16: 1, fp16: 2, fp32: 3), each plane product is exact in the
// fp32 accumulator.  One wave: 16 rows of dS x 16 columns of dq.
// ---------------------------------------------------------------------------
// x as the sum of PL bf16 values: cut off, not rounded, so that each plane
// holds the next 8 significant bits and nothing overflows; infinities and NaN
// are in the first plane alone (a NaN keeps a bit that survives the cut)
template <int PL>
__device__ __forceinline__ void split_planes(const float (&x)[8], bf16x8 (&pl)[PL]) {
  u32x4 w[PL];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t b[2][PL];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float r = x[2 * k + e];
      if (PL > 1 && !(fabsf(r) < __builtin_inff())) {
        b[e][0] = r != r ? 0x7FC00000u : __float_as_uint(r);
        r = 0.f;
      } else {
        b[e][0] = __float_as_uint(r) & 0xFFFF0000u;
        r -= __uint_as_float(b[e][0]);
      }
#pragma unroll
      for (int q = 1; q < PL; ++q) {
        b[e][q] = __float_as_uint(r) & 0xFFFF0000u;
        r -= __uint_as_float(b[e][q]);
      }
    }
#pragma unroll
    for (int q = 0; q < PL; ++q) w[q][k] = (b[0][q] >> 16) | b[1][q];
  }
#pragma unroll
  for (int q = 0; q < PL; ++q) pl[q] = __builtin_bit_cast(bf16x8, w[q]);
}

template <int DT, int DQ>
__global__ __launch_bounds__(64) void k_cat_dq(const void* ds, int64_t m, int64_t lds, int64_t n, const uint8_t* codes,
                                               const uint8_t* scales, int d, int nkb, void* dq, int col_tiles) {
  using namespace b8;
  constexpr int PL = DT == TT_BF16 ? 1 : DT == TT_F16 ? 2 : 3;
  const int l = lane_id(), r = l & 15, g = l >> 4;
  const int64_t m0 = (int64_t)(blockIdx.x / col_tiles) * 16;
  const int c0 = (int)(blockIdx.x % col_tiles) * 16;
  const int64_t row = min(m0 + r, m - 1);
  f32x4 acc = zero4();
  for (int64_t n0 = 0; n0 < n; n0 += 32) {
    float x[8], c[8];
    const int64_t nn = n0 + 8 * g;
    ld8n<DT>(ds, row * lds + nn, (int)max((int64_t)0, min((int64_t)8, n - nn)), x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t cr = min(nn + e, n - 1);
      float v[4];
      decode4((uint32_t)codes[(cr * nkb) * BLK + c0 + r], scale_of(scales[cr * nkb + c0 / BLK]), v);
      c[e] = nn + e < n ? v[0] : 0.f;
    }
    bf16x8 a[PL], b[1];
    split_planes<PL>(x, a);
    split_planes<1>(c, b);
#pragma unroll
    for (int q = PL - 1; q >= 0; --q) acc = mfma_bf16(a[q], b[0], acc);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t i = m0 + 4 * g + e;
    if (i < m && c0 + r < d) st1<DQ>(dq, i * d + c0 + r, acc[e]);
  }
}

}  // namespace tt
