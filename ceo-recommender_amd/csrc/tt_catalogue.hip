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
// owner to its own place + 1 (k_cat_own), then only the owner writes
// (k_cat_write), and every mention puts the word back to zero (k_cat_disown):
// three launches, 100000 of a million rows of 256 in bf16 28 us.
__global__ __launch_bounds__(256) void k_cat_own(CatRows r, int64_t m, int32_t* owner) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < m; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t c = r.rows[i];
    if (cat_row_ok(r, c)) atomicMax(owner + c, (int32_t)i + 1);
  }
}

// 16 lanes take up to CAT_UNIT blocks of a row (blockIdx.y: which ones), 8
// values each: all loads first, one row number and one owner for all of them.
// Bound by memory: a million rows of 256 in bf16 written 152 us (5.1 TB/s),
// read 124 us (6.3 TB/s); a division a block instead of blockIdx.y 158, 135 us
constexpr int CAT_UNIT = 2;
template <int DT>
__global__ __launch_bounds__(256) void k_cat_write(const void* x, int64_t m, int64_t ldx, int d, int nkb, CatRows r,
                                                   uint8_t* codes, uint8_t* scales, int32_t* owner) {
  using namespace b8;
  const int lane = (int)threadIdx.x % LANES, kb0 = (int)blockIdx.y * CAT_UNIT;
  for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LANES; i < m;
       i += (int64_t)gridDim.x * blockDim.x / LANES) {
    const int64_t c = cat_row(r, i);
    if (!cat_row_ok(r, c)) continue;
    if (owner && owner[c] != (int32_t)i + 1) continue;
    float v[CAT_UNIT][8];
#pragma unroll
    for (int b = 0; b < CAT_UNIT; ++b) {
      const int k = (kb0 + b) * BLK + lane * 8;
      ld8n<DT>(x, i * ldx + k, max(0, min(8, d - k)), v[b]);
    }
#pragma unroll
    for (int b = 0; b < CAT_UNIT; ++b)
      if (kb0 + b < nkb) {
        uint32_t byte;
        const u32x2 w = encode8(v[b], byte);
        __builtin_memcpy(codes + (c * nkb + kb0 + b) * BLK + lane * 8, &w, 8);
        if (lane == 0) scales[c * nkb + kb0 + b] = (uint8_t)byte;
      }
  }
}
__global__ __launch_bounds__(256) void k_cat_disown(CatRows r, int64_t m, int32_t* owner) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < m; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t c = r.rows[i];
    if (cat_row_ok(r, c)) owner[c] = 0;
  }
}

// Up to CAT_FEW rows in one launch: every workgroup holds all row numbers in LDS
// and the 16 lanes of a block look for a later mention of theirs (calls one after
// the other against three launches, us, 60 values in fp32: 10 rows 3.4 / 6.2, 333
// 4.2 / 6.7, 1000 6.5 / 7.2)
constexpr int CAT_FEW = 1024;
template <int DT>
__global__ __launch_bounds__(256) void k_cat_write_few(const void* x, int m, int64_t ldx, int d, int nkb, CatRows r,
                                                       uint8_t* codes, uint8_t* scales) {
  using namespace b8;
  __shared__ int64_t rows[CAT_FEW];
  for (int i = (int)threadIdx.x; i < m; i += 256) rows[i] = r.rows[i];
  __syncthreads();
  const int u = (int)(blockIdx.x * 256 + threadIdx.x) / LANES, lane = (int)threadIdx.x % LANES;
  if (u >= m * nkb) return;
  const int i = u / nkb, kb = u % nkb;
  const int64_t c = rows[i];
  if (!cat_row_ok(r, c)) return;
  bool later = false;
  for (int j = i + 1 + lane; j < m; j += LANES) later |= rows[j] == c;
  const uint64_t any = __ballot(later) >> (threadIdx.x & 48) & 0xFFFFu;
  if (any) return;
  const int k = kb * BLK + lane * 8;
  float v[8];
  ld8n<DT>(x, i * ldx + k, max(0, min(8, d - k)), v);
  uint32_t byte;
  const u32x2 w = encode8(v, byte);
  __builtin_memcpy(codes + (c * nkb + kb) * BLK + lane * 8, &w, 8);
  if (lane == 0) scales[c * nkb + kb] = (uint8_t)byte;
}

template <int DT>
__global__ __launch_bounds__(256) void k_cat_read(const uint8_t* codes, const uint8_t* scales, CatRows r, int64_t m,
                                                  int d, int nkb, void* out, int64_t ldo) {
  using namespace b8;
  const int lane = (int)threadIdx.x % LANES, kb0 = (int)blockIdx.y * CAT_UNIT;
  for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LANES; i < m;
       i += (int64_t)gridDim.x * blockDim.x / LANES) {
    const int64_t c = cat_row(r, i);
    u32x2 w[CAT_UNIT];
    uint32_t byte[CAT_UNIT];
    const bool ok = cat_row_ok(r, c);
#pragma unroll
    for (int b = 0; b < CAT_UNIT; ++b) {
      w[b] = (u32x2){0u, 0u};
      byte[b] = 127u;
      if (ok && kb0 + b < nkb) {
        __builtin_memcpy(&w[b], codes + (c * nkb + kb0 + b) * BLK + lane * 8, 8);
        byte[b] = scales[c * nkb + kb0 + b];
      }
    }
#pragma unroll
    for (int b = 0; b < CAT_UNIT; ++b) {
      const int k = (kb0 + b) * BLK + lane * 8;
      float v[8];
      decode8(w[b], scale_of(byte[b]), v);
      st8n<DT>(out, i * ldo + k, max(0, min(8, d - k)), v);
    }
  }
}

// ---------------------------------------------------------------------------
// scores = Q^ C^^T.  Lane l supplies 32 bytes of operand row l & 15 for a block
// of 128: 16-byte chunks l >> 4 and (l >> 4) + 4 of the row (the same for both
// operands, so this order of k is right; a load then takes 64 bytes of a row);
// C: lane l holds C[row = 4 (l >> 4) + reg][column = l & 15].
//
// Both operands are decoded to bf16, exactly, for v_mfma_f32_16x16x32_bf16,
// whose sums measured 8e-8 of the result in the 2-norm.  The 8-bit matrix
// instructions, scaled ones and others, are no sums in 32 bits: they cut the
// products of one instruction off below the largest of them (over all e4m3
// values a sum of 128 is off by up to 2^-11 of its largest product, 5e-5 in the
// 2-norm), which products that cancel leave in the result whatever its type.
// They took 420 us where this takes 550 (8192 x 100000 x 256 in bf16), 17.6 /
// 23.3 (513 x 20011 x 512), 39.1 / 41.8 (37 x 1000003 x 128), 277 / 271 (16384 x
// 32771 x 128).
// ---------------------------------------------------------------------------
typedef int i32x8 __attribute__((ext_vector_type(8)));

// 8 codes and their block's scale -> bf16, exact
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t lo, uint32_t hi, float s) {
  u32x4 w;
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true));
  w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false));
  w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true));
  return __builtin_bit_cast(bf16x8, w);
}
__device__ __forceinline__ f32x4 mfma_block(const i32x8& a, const i32x8& b, f32x4 c, int sa, int sb) {
  const float fa = b8::scale_of((uint32_t)sa), fb = b8::scale_of((uint32_t)sb);
#pragma unroll
  for (int h = 0; h < 4; ++h)
    c = mfma_bf16(codes_to_bf16((uint32_t)a[2 * h], (uint32_t)a[2 * h + 1], fa),
                  codes_to_bf16((uint32_t)b[2 * h], (uint32_t)b[2 * h + 1], fb), c);
  return c;
}

__device__ __forceinline__ i32x8 frag_of(const u32x4& lo, const u32x4& hi) {
  return (i32x8){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
// from the 128 bytes of a row at p (16-byte aligned)
__device__ __forceinline__ i32x8 row_frag(const uint8_t* p, int g) {
  return frag_of(*reinterpret_cast<const u32x4*>(p + 16 * g), *reinterpret_cast<const u32x4*>(p + 16 * g + 64));
}

// LDS image of 128-byte rows (one block of codes each): 16-byte chunk c of row
// r lies at chunk c ^ (r & 7), so that 8 lanes that read one chunk of 8
// consecutive rows touch all 32 banks once.
constexpr int ROWB = TT_BLOCK;
__device__ __forceinline__ int lds_chunk(int row, int c) { return row * ROWB + ((c ^ (row & 7)) << 4); }
__device__ __forceinline__ i32x8 lds_frag(const uint8_t* s, int row, int g) {
  return frag_of(*reinterpret_cast<const u32x4*>(s + lds_chunk(row, g)),
                 *reinterpret_cast<const u32x4*>(s + lds_chunk(row, g + 4)));
}
// loads straight into LDS have arrived
__device__ __forceinline__ void wait_lds_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A wave's tile of 16 QT queries x 16 IT catalogue rows, stored row by row:
// lane (r, g) holds 4 consecutive columns of row r; it is turned in the wave's
// own LDS so that 16-byte pieces of whole rows go out (pieces at any address:
// rows of odd length start anywhere).
template <int DT, int IT, int QT> constexpr int tile_lds() { return 16 * QT * (16 * IT * b8::Elem<DT>::SIZE + 16); }
// WHOLE: all 16 IT columns exist and 64 rows of the result span less than 2 GiB
template <int DT, int IT, int QT, bool WHOLE>
__device__ __forceinline__ void store_tile(uint8_t* so, const f32x4 (&acc)[IT][QT], void* out, int64_t m0, int64_t m,
                                           int64_t n0, int64_t n) {
  using namespace b8;
  constexpr int ES = Elem<DT>::SIZE, LDO = 16 * IT * ES + 16;
  constexpr int PER = 16 / ES, LPR = 16 * IT / PER;  // values of a piece, pieces of a row
  const int l = lane_id(), r = l & 15, g = l >> 4;
#pragma unroll
  for (int j = 0; j < QT; ++j)
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      uint8_t* at = so + (16 * j + r) * LDO + (16 * i + 4 * g) * ES;
      const f32x4 v = acc[i][j];
      if constexpr (DT == TT_F32)
        *reinterpret_cast<f32x4*>(at) = v;
      else if constexpr (DT == TT_BF16)
        *reinterpret_cast<u32x2*>(at) = (u32x2){pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])};
      else
        *reinterpret_cast<u32x2*>(at) = (u32x2){float_to_half_bits(v[0]) | (uint32_t)float_to_half_bits(v[1]) << 16,
                                                float_to_half_bits(v[2]) | (uint32_t)float_to_half_bits(v[3]) << 16};
    }
  __builtin_amdgcn_wave_barrier();
  const int rows = (int)min((int64_t)(16 * QT), m - m0), cols = (int)min((int64_t)(16 * IT), n - n0);
  uint8_t* const base = (uint8_t*)out + (m0 * n + n0) * ES;
#pragma unroll
  for (int k = 0; k < (16 * QT * LPR + 63) / 64; ++k) {
    const int u = k * 64 + l;
    const bool piece = 16 * QT * LPR % 64 == 0 || u < 16 * QT * LPR;
    const int row = piece ? u / LPR : 0, c = (u % LPR) * PER;
    const uint8_t* from = so + row * LDO + c * ES;
    if constexpr (WHOLE) {
      // no branch: the loop over tiles then knows how many stores follow the
      // next tile's loads and waits for the loads alone
      const uint32_t off = piece && row < rows ? (uint32_t)row * (uint32_t)(n * ES) + (uint32_t)(c * ES) : 0x80000000u;
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(base, (short)0, 0x7FFFFFFF, 0x00020000);
      __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const u32x4*>(from), rs, (int)off, 0, 0);
    } else if (piece && row < rows && c < cols) {
      uint8_t* to = base + ((int64_t)row * n + c) * ES;
      if (c + PER <= cols) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(from);
        __builtin_memcpy(to, &v, 16);
      } else {
        for (int e = 0; e < cols - c; ++e) __builtin_memcpy(to + e * ES, from + e * ES, ES);
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
}

// Up to 64 queries, bound by the catalogue's bytes: a wave keeps 16 QT queries
// in registers and walks over the catalogue, 16 IT rows at a time, straight
// from global memory: no barrier, and the next rows' loads fly while this tile
// is stored.  The 4 waves of a workgroup take neighbouring row groups, so that
// a query's results go out in pieces of 64 IT values.  Measured, calls back to
// back (the codes stay in the last-level cache): 1 x 1000003 x 128 24.4 us, 16 x
// 1000003 x 128 29.6 us, 1 x 100000 x 256 8.1 us.  For more queries the tiles below
// are faster (8192 x 100000 x 256 on the 8-bit instructions: 776 against 420 us:
// every wave reads the catalogue through L2 again).
struct StreamArgs {
  const void* q;            // raw queries (ENC) or their codes
  const uint8_t* qs;        // their scale bytes (not ENC)
  const uint8_t *codes, *scales;
  void* out;
  int64_t m, n, ldq;
  int d, nkb, q_dtype;
  int64_t strips, per;          // workgroups; those of an XCD
};

// NKB: blocks a row, the queries encoded here and held in registers; 0: any number, with the queries' codes from the
// workspace read again for every tile
template <int DT, int IT, int QT, int NKB>
__global__ __launch_bounds__(256, QT == 4 ? 2 : 1) void k_cat_stream(StreamArgs a) {
  using namespace b8;
  constexpr bool ENC = NKB > 0;
  constexpr int KB = ENC ? NKB : 1;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * tile_lds<DT, IT, QT>()];
  __shared__ __attribute__((aligned(16))) uint8_t enc[ENC ? 16 * QT * KB * (ROWB + 1) : 16];  // ENC: the queries' codes, scale bytes
  const int l = lane_id(), w = wave_id(), r = l & 15, g = l >> 4;
  uint8_t* const so = lds + w * tile_lds<DT, IT, QT>();
  const int64_t strip = (int64_t)(blockIdx.x & 7) * a.per + (blockIdx.x >> 3);
  if (strip >= a.strips) return;
  const int64_t n = a.n;
  const int nkb = ENC ? NKB : a.nkb;
  // this strip's groups of 64 IT rows
  const int64_t groups = (n + 64 * IT - 1) / (64 * IT);
  const int64_t g0 = groups * strip / a.strips, g1 = groups * (strip + 1) / a.strips;

  // the first rows' loads go out before the queries are read and encoded
  i32x8 x[KB][IT];
  int sa[KB][IT];
  auto load = [&](int64_t n0) {
    const int last = (int)min((int64_t)(16 * IT), n - n0) - 1;
    const uint8_t* c0 = a.codes + n0 * (KB * ROWB);
    const uint8_t* s0 = a.scales + n0 * KB;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const uint32_t row = (uint32_t)min(16 * i + r, last);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        x[kb][i] = row_frag(c0 + (row * KB + kb) * ROWB, g);
        sa[kb][i] = s0[row * KB + kb];
      }
    }
  };
  int64_t n0 = (g0 * 4 + w) * 16 * IT;
  const int64_t end = min(n, g1 * 64 * IT);
  if (ENC && n0 < end) load(n0);

  const uint8_t* qrow[QT];
  const uint8_t* qsrow[QT];
  i32x8 b[KB][QT];
  int sb[KB][QT];
  if constexpr (ENC) {
    // the workgroup encodes its queries once, 16 lanes a block
    for (int u = (int)threadIdx.x / LANES; u < a.m * KB; u += 256 / LANES) {
      const int i = u / KB, kb = u % KB, lane = (int)threadIdx.x % LANES, k = kb * BLK + lane * 8, live = max(0, min(8, a.d - k));
      float v[8];
      if (a.q_dtype == TT_F32)
        ld8n<TT_F32>(a.q, i * a.ldq + k, live, v);
      else if (a.q_dtype == TT_BF16)
        ld8n<TT_BF16>(a.q, i * a.ldq + k, live, v);
      else
        ld8n<TT_F16>(a.q, i * a.ldq + k, live, v);
      uint32_t byte;
      *reinterpret_cast<u32x2*>(enc + u * ROWB + lane * 8) = encode8(v, byte);
      if (lane == 0) enc[16 * QT * KB * ROWB + u] = (uint8_t)byte;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      const int row = min(16 * j + r, (int)a.m - 1);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        b[kb][j] = row_frag(enc + (row * KB + kb) * ROWB, g);
        sb[kb][j] = enc[16 * QT * KB * ROWB + row * KB + kb];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      const int64_t at = min((int64_t)(16 * j + r), a.m - 1);
      qrow[j] = (const uint8_t*)a.q + at * nkb * ROWB;
      qsrow[j] = a.qs + at * nkb;
    }
  }

  if constexpr (ENC) {
    f32x4 acc[IT][QT];
    auto multiply = [&]() {
#pragma unroll
      for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < QT; ++j) acc[i][j] = zero4();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
          for (int j = 0; j < QT; ++j)
            acc[i][j] = mfma_block(x[kb][i], b[kb][j], acc[i][j], sa[kb][i], sb[kb][j]);
    };
    // whole tiles first; addresses of the one after the last stay inside the catalogue
    const int64_t whole = n * Elem<DT>::SIZE * 64 < 0x7FFFFFFF ? end - 16 * IT : -1;
    while (n0 <= whole) {
      multiply();
      const int64_t at = n0;
      n0 += 64 * IT;
      load(min(n0, n - 1));  // in flight while this tile is stored
      store_tile<DT, IT, QT, true>(so, acc, a.out, 0, a.m, at, n);
    }
    while (n0 < end) {
      multiply();
      store_tile<DT, IT, QT, false>(so, acc, a.out, 0, a.m, n0, n);
      n0 += 64 * IT;
      if (n0 < end) load(n0);
    }
  } else {
    for (int64_t u = g0; u < g1; ++u) {
      const int64_t n0 = (u * 4 + w) * 16 * IT;
      if (n0 >= n) break;
      const int last = (int)min((int64_t)(16 * IT), n - n0) - 1;
      const uint8_t* c0 = a.codes + n0 * nkb * ROWB;
      const uint8_t* s0 = a.scales + n0 * nkb;
      f32x4 acc[IT][QT];
#pragma unroll
      for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < QT; ++j) acc[i][j] = zero4();
      for (int kb = 0; kb < nkb; ++kb) {
        i32x8 x[IT], y[QT];
        int sx[IT], sy[QT];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int64_t row = min(16 * i + r, last);
          x[i] = row_frag(c0 + (row * nkb + kb) * ROWB, g);
          sx[i] = s0[row * nkb + kb];
        }
#pragma unroll
        for (int j = 0; j < QT; ++j) {
          y[j] = row_frag(qrow[j] + (int64_t)kb * ROWB, g);
          sy[j] = qsrow[j][kb];
        }
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
          for (int j = 0; j < QT; ++j) acc[i][j] = mfma_block(x[i], y[j], acc[i][j], sx[i], sy[j]);
      }
      store_tile<DT, IT, QT, false>(so, acc, a.out, 0, a.m, n0, n);
    }
  }
}

// a wave's 64 x 64 results, STORE_J 16-query tiles at a time
template <int DT> constexpr int STORE_J = DT == TT_F32 ? 2 : 4;
template <int DT>
__device__ __forceinline__ void store_wave(uint8_t* so, const f32x4 (&acc)[4][4], void* out, int64_t m0, int64_t m,
                                           int64_t n0, int64_t n) {
  constexpr int J = STORE_J<DT>;
#pragma unroll
  for (int j0 = 0; j0 < 4; j0 += J) {
    f32x4 y[4][J];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) y[i][j] = acc[i][j0 + j];
    store_tile<DT, 4, J, false>(so, y, out, m0 + 16 * j0, m, n0, n);
  }
}

// Many queries: one workgroup a tile of 128 queries x 128 catalogue rows, a
// wave 64 x 64 of it, a block of 128 values staged in LDS at a time.  Nothing is
// fetched ahead: three workgroups a CU (164 registers a lane, 36 KB) cover each
// other's loads and stores (four, with 92 bytes a lane in scratch: 829 for 543 us
// at 8192 x 100000 x 256 in bf16).
constexpr int CT_M = 128, CT_N = 128;

// Tile of workgroup `id` of 8 * per: XCD x runs workgroups x, x + 8, ... and
// takes the x-th eighth of the tiles, in panels of `width` column tiles walked
// over all row tiles: its L2 holds a panel's catalogue rows (512 KB at most)
// and meets every query once a panel.  Wide panels also write long pieces of
// the same rows at a time.  8 / 16 / 32 / 64 column tiles, us, bf16: 16384 x 32771 x
// 128 319 / 321 / 272 / 283, 8192 x 100000 x 256 545 / 534 / 585 / 581.
__device__ __forceinline__ bool cat_tile(int64_t id, int64_t per, int64_t mt, int64_t nt, int width, int64_t& tm,
                                         int64_t& tn) {
  const int64_t t = (id & 7) * per + (id >> 3);
  if (t >= mt * nt) return false;
  const int64_t panel = (int64_t)width * mt, p = t / panel, in = t - p * panel;
  const int64_t cols = min((int64_t)width, nt - p * width);  // the last panel may be narrower
  tn = p * width + in % cols;
  tm = in / cols;
  return true;
}

template <int DT>
__global__ __launch_bounds__(256, 3) void k_cat_scores(
    const uint8_t* __restrict__ q, const uint8_t* __restrict__ qs, int64_t m, const uint8_t* __restrict__ codes,
    const uint8_t* __restrict__ scales, int64_t n, int nkb, void* out, int64_t mt, int64_t nt, int64_t per, int width) {
  using namespace b8;
  constexpr int SO = 4 * tile_lds<DT, 4, STORE_J<DT>>();
  __shared__ __attribute__((aligned(128))) uint8_t lds[SO > 2 * 128 * ROWB + 256 ? SO : 2 * 128 * ROWB + 256];
  uint8_t* const sc = lds;               // catalogue rows
  uint8_t* const sq = lds + CT_N * ROWB; // queries
  const int l = lane_id(), w = wave_id(), r = l & 15, g = l >> 4;
  int64_t tm, tn;
  if (!cat_tile(blockIdx.x, per, mt, nt, width, tm, tn)) return;
  const int64_t m0 = tm * CT_M, n0 = tn * CT_N;
  const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
  const int rows_q = (int)min((int64_t)CT_M, m - m0), rows_c = (int)min((int64_t)CT_N, n - n0);

  // staging: 8 rows a wave and instruction, wave w takes rows 32 w .. 32 w + 31
  // of both operands; loads past the last row bring zeros
  const int64_t kp = (int64_t)nkb * ROWB;
  const uint32_t off = (uint32_t)((l >> 3) * kp + (((l & 7) ^ (l >> 3)) << 4));
  auto stage = [&](const uint8_t* from, int rows, uint8_t* to) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int first = 32 * w + 8 * i;
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(from + first * kp), (short)0,
                                                        (int)(max(0, rows - first) * kp), 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(to + first * ROWB), 16,
                                               (int)off, 0, 0, 0);
    }
  };
  const uint8_t *gc = codes + n0 * kp, *gq = q + m0 * kp;
  // thread t brings the scale byte of catalogue row t or of query t - 128
  const int srow = (int)threadIdx.x % 128;
  const uint8_t* gs = (int)threadIdx.x < 128 ? scales + (n0 + min(srow, rows_c - 1)) * nkb : qs + (m0 + min(srow, rows_q - 1)) * nkb;
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = zero4();

  for (int kb = 0; kb < nkb; ++kb) {
    stage(gc + kb * ROWB, rows_c, sc);
    stage(gq + kb * ROWB, rows_q, sq);
    lds[2 * 128 * ROWB + threadIdx.x] = gs[kb];
    wait_lds_loads();
    __syncthreads();
    i32x8 a[4];
    int sa[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = lds_frag(sc, wn + 16 * i + r, g);
      sa[i] = lds[2 * 128 * ROWB + wn + 16 * i + r];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const i32x8 b = lds_frag(sq, wm + 16 * j + r, g);
      const int sb = lds[2 * 128 * ROWB + 128 + wm + 16 * j + r];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][j] = mfma_block(a[i], b, acc[i][j], sa[i], sb);
    }
    __syncthreads();
  }

  store_wave<DT>(lds + w * tile_lds<DT, 4, STORE_J<DT>>(), acc, out, m0 + wm, m, n0 + wn, n);
}

// ---------------------------------------------------------------------------
// dq = dS C^ on v_mfma_f32_16x16x32_bf16: C^ is exact in bf16, dS is split into
// bf16 planes that hold it exactly (bf16: 1, fp16: 2, fp32: 3), each product
// is exact in the fp32 accumulator.
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

struct DqArgs {
  const void* ds;
  int64_t m, lds, n;
  const uint8_t *codes, *scales;
  int d, nkb;
  void* out;               // dq, or the parts [splits][m][d] in fp32
  int64_t mt, splits, per; // row blocks, parts of the catalogue, workgroups of an XCD
  int groups;              // column groups of 16 CT
  int64_t part_steps;      // steps of DQ_STEP catalogue rows in a part
};

// 8 consecutive values of a row of dS as they lie in memory
template <int DT> struct DsFrag {
  u32x4 v[DT == TT_F32 ? 2 : 1];
};
// The same as it was loaded.  ODD (16-bit values, rows an odd number of them
// apart, the first on a 4-byte boundary): loads at 2-byte addresses take longer
// (16384 x 32771 x 128 421 us in bf16, 495 in fp16), so a lane loads the 5 words
// that hold its 8 values and shifts later (324, 427).  The words reach one value
// past the 8 and, in odd rows, one before: both are in the array, since the
// steps that load this way end before the row does.
template <int DT, bool ODD> struct DsLoad {
  u32x4 v[DT == TT_F32 ? 2 : 1];
  uint32_t next;
};
template <int DT> struct DsLoad<DT, false> {
  u32x4 v[DT == TT_F32 ? 2 : 1];
};
template <int DT, bool ODD>
__device__ __forceinline__ void load_ds(const uint8_t* row, int64_t at, DsLoad<DT, ODD>& to) {
  const uint8_t* p = row + at * b8::Elem<DT>::SIZE;
  if constexpr (ODD) {
    const bool half = ((uintptr_t)row & 2) != 0;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p - (half ? 2 : 0));
    __builtin_memcpy(&to.v[0], w, 16);
    to.next = w[half ? 4 : 3];
  } else {
    __builtin_memcpy(&to.v, p, sizeof(to.v));
  }
}
template <int DT, bool ODD>
__device__ __forceinline__ DsFrag<DT> ds_values(const DsLoad<DT, ODD>& x, bool half) {
  DsFrag<DT> f;
  if constexpr (ODD) {
    const uint32_t sh = half ? 16u : 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      f.v[0][k] = __builtin_amdgcn_alignbit(k < 3 ? x.v[0][k + 1] : x.next, x.v[0][k], sh);
  } else {
    __builtin_memcpy(&f, &x, sizeof(f));
  }
  return f;
}
// one by one, zeros from `live` on
template <int DT>
__device__ __forceinline__ DsFrag<DT> load_ds_last(const uint8_t* row, int64_t at, int live) {
  constexpr int ES = b8::Elem<DT>::SIZE;
  DsFrag<DT> f;
  const uint8_t* p = row + at * ES;
#pragma unroll
  for (int w = 0; w < 2 * ES; ++w) {
    uint32_t x = 0;
    if constexpr (ES == 4) {
      if (w < live) __builtin_memcpy(&x, p + 4 * w, 4);
    } else {
      uint16_t lo = 0, hi = 0;
      if (2 * w < live) __builtin_memcpy(&lo, p + 4 * w, 2);
      if (2 * w + 1 < live) __builtin_memcpy(&hi, p + 4 * w + 2, 2);
      x = lo | (uint32_t)hi << 16;
    }
    f.v[w / 4][w % 4] = x;
  }
  return f;
}
template <int DT, int PL>
__device__ __forceinline__ void ds_planes(const DsFrag<DT>& f, bf16x8 (&a)[PL]) {
  if constexpr (DT == TT_BF16) {
    a[0] = __builtin_bit_cast(bf16x8, f.v[0]);
  } else {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = DT == TT_F32 ? __uint_as_float(f.v[e / 4][e % 4])
                          : b8::half_bits_to_float((uint16_t)(f.v[0][e / 2] >> (16 * (e & 1))));
    split_planes<PL>(x, a);
  }
}

// Bound by dS's bytes up to 128 columns, then by what LDS hands the waves.
// Measured in bf16: 16384 x 32768 x 128 238 us (4.5 TB/s), x 32771 324-356 us, 8192
// x 100000 x 256 540 us (3.0 TB/s; 16 rows a wave read LDS twice as often, 649 us);
// in fp16 358, 427, 890 us; in fp32 8192 x 32768 x 128 276 us.
// One workgroup: 16 RT WM rows of dS against a part of the catalogue, 16 CT
// columns of dq in its waves' accumulators.  A step of DQ_STEP catalogue rows
// is decoded once into LDS as bf16 [row][column] and read back transposed; the
// next step's codes and dS values are on their way meanwhile.  WM waves take
// different rows; with WM = 1 (up to 16 rows) four share the rows and take
// different thirty-twos of a step's catalogue rows, and add up at the end.
constexpr int DQ_ROW_PAD = 32;  // bytes: 4 rows of a transposed read in distinct banks
template <int WM> constexpr int DQ_STEP = WM == 1 ? 128 : 64;
template <int CT, int WM> constexpr int dq_lds() {
  const int stage = 2 * DQ_STEP<WM> * (32 * CT + DQ_ROW_PAD), sum = WM == 1 ? 4 * 16 * 16 * CT * 4 : 0;
  return stage > sum ? stage : sum;
}
template <int DT, int DQ, int CT, int RT, int WM, bool ODD>
__global__ __launch_bounds__(256, 2) void k_cat_dq(DqArgs a) {
  using namespace b8;
  constexpr int PL = DT == TT_BF16 ? 1 : DT == TT_F16 ? 2 : 3;
  constexpr int STEP = DQ_STEP<WM>;
  constexpr int KS = WM == 1 ? 1 : STEP / 32;  // 32-row products of a wave in a step
  constexpr int RS = 32 * CT + DQ_ROW_PAD;                 // bytes of a row in LDS
  constexpr int CH = STEP * CT / 256;                      // 16-code pieces a thread decodes in a step
  extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
  const int l = lane_id(), w = wave_id(), r = l & 15, g = l >> 4;
  const int64_t id = (int64_t)(blockIdx.x & 7) * a.per + (blockIdx.x >> 3);
  const int64_t row_blocks = a.mt * a.groups;
  if (id >= row_blocks * a.splits) return;
  const int64_t part = id / row_blocks, in = id % row_blocks;
  const int col0 = (int)(in % a.groups) * 16 * CT;
  const int64_t m0 = (in / a.groups) * (16 * RT * WM) + (WM == 1 ? 0 : w * 16 * RT);
  const int64_t n = a.n, n_from = part * a.part_steps * STEP, n_to = min(n, n_from + a.part_steps * STEP);
  const int64_t kp = (int64_t)a.nkb * ROWB;

  const uint8_t* row[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) row[i] = (const uint8_t*)a.ds + min(m0 + 16 * i + r, a.m - 1) * a.lds * Elem<DT>::SIZE;
  const int ks0 = WM == 1 ? w : 0;  // this wave's first 32 rows of a step

  // this thread's 16-code pieces of a step, as offsets from the step's first row
  const uint8_t* const codes = a.codes + col0;
  uint32_t co[CH], so[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int u = c * 256 + (int)threadIdx.x, cr = u / CT;
    const int cc = min((u % CT) * 16, (int)kp - 16 - col0);  // past the row's end: any codes, the columns are not stored
    co[c] = (uint32_t)(cr * kp + cc);
    so[c] = (uint32_t)(cr * a.nkb + (col0 + cc) / ROWB);
  }
  struct Codes {
    u32x4 v[CH];
    uint32_t byte[CH];
  };
  Codes code[2];
  DsLoad<DT, ODD> ds[2][RT][KS];
  auto fetch_codes = [&](int64_t n0, Codes& to) {
    const uint8_t* c0 = codes + n0 * kp;
    const uint8_t* s0 = a.scales + n0 * a.nkb;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      to.v[c] = *reinterpret_cast<const u32x4*>(c0 + co[c]);
      to.byte[c] = s0[so[c]];
    }
  };
  auto fetch_ds = [&](int64_t n0, DsLoad<DT, ODD> (&to)[RT][KS]) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int k = 0; k < KS; ++k) load_ds<DT, ODD>(row[i], n0 + 32 * (ks0 + k) + 8 * g, to[i][k]);
  };
  // the catalogue's last step, shorter than the others: zeros past the end
  auto fetch_last = [&](int64_t n0, Codes& cd, DsFrag<DT> (&to)[RT][KS]) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const bool live = n0 + (c * 256 + (int)threadIdx.x) / CT < n;
      cd.v[c] = (u32x4){0u, 0u, 0u, 0u};
      cd.byte[c] = 127u;
      if (live) {
        cd.v[c] = *reinterpret_cast<const u32x4*>(codes + n0 * kp + co[c]);
        cd.byte[c] = a.scales[n0 * a.nkb + so[c]];
      }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int64_t at = n0 + 32 * (ks0 + k) + 8 * g;
        to[i][k] = load_ds_last<DT>(row[i], at, (int)max((int64_t)0, min((int64_t)8, n - at)));
      }
  };
  auto decode = [&](const Codes& cd, uint8_t* to) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int u = c * 256 + (int)threadIdx.x, cr = u / CT, cc = (u % CT) * 16;
      const float s = scale_of(cd.byte[c]);
      *reinterpret_cast<bf16x8*>(to + cr * RS + cc * 2) = codes_to_bf16(cd.v[c][0], cd.v[c][1], s);
      *reinterpret_cast<bf16x8*>(to + cr * RS + cc * 2 + 16) = codes_to_bf16(cd.v[c][2], cd.v[c][3], s);
    }
  };
  f32x4 acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[i][c] = zero4();
  auto multiply = [&](const uint8_t* from, auto values) {
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      bf16x8 f[RT][PL];
#pragma unroll
      for (int i = 0; i < RT; ++i) ds_planes<DT, PL>(values(i, k), f[i]);
      const uint8_t* at = from + (32 * (ks0 + k) + 8 * g + (r >> 2)) * RS + (r & 3) * 8;
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const bf16x8 b = tr_frag(reinterpret_cast<const uint16_t*>(at + 32 * c),
                                 reinterpret_cast<const uint16_t*>(at + 32 * c + 4 * RS));
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int q = PL - 1; q >= 0; --q) acc[i][c] = mfma_bf16(f[i][q], b, acc[i][c]);
      }
    }
  };

  uint8_t* const stage[2] = {lds, lds + STEP * RS};
  auto use = [&](int p) {
    multiply(stage[p], [&](int i, int k) { return ds_values<DT, ODD>(ds[p][i][k], ((uintptr_t)row[i] & 2) != 0); });
  };
  // steps that end inside the row (ODD: before its end)
  const int64_t whole = n_from + max((int64_t)0, min(n_to, ODD ? n - 1 : n) - n_from) / STEP * STEP;
  if (n_from < whole) {
    // two steps a round, so that each buffer has a name.  A buffer is filled
    // again right after its use: dS two steps ahead, codes three (past the
    // part's end the last step is fetched again, unused)
    const int64_t end = whole - STEP;
    fetch_codes(n_from, code[0]);
    fetch_codes(min(n_from + STEP, end), code[1]);
    fetch_ds(n_from, ds[0]);
    fetch_ds(min(n_from + STEP, end), ds[1]);
    decode(code[0], stage[0]);
    fetch_codes(min(n_from + 2 * STEP, end), code[0]);
    for (int64_t n0 = n_from;; n0 += 2 * STEP) {
      __syncthreads();
      use(0);
      if (n0 + STEP >= whole) break;
      fetch_ds(min(n0 + 2 * STEP, end), ds[0]);
      decode(code[1], stage[1]);
      fetch_codes(min(n0 + 3 * STEP, end), code[1]);
      __syncthreads();
      use(1);
      if (n0 + 2 * STEP >= whole) break;
      fetch_ds(min(n0 + 3 * STEP, end), ds[1]);
      decode(code[0], stage[0]);
      fetch_codes(min(n0 + 4 * STEP, end), code[0]);
    }
  }
  if (whole < n_to) {
    DsFrag<DT> last[RT][KS];
    __syncthreads();
    fetch_last(whole, code[0], last);
    decode(code[0], stage[0]);
    __syncthreads();
    multiply(stage[0], [&](int i, int k) { return last[i][k]; });
  }

  if constexpr (WM == 1) {  // the four waves' sums, in wave order
    __syncthreads();
    float* const sum = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[((w * 16 + 4 * g + e) * CT + c) * 16 + r] = acc[0][c][e];
    __syncthreads();
    constexpr int W = 16 * 16 * CT;
    for (int u = (int)threadIdx.x; u < W; u += 256) {
      const float v = ((sum[u] + sum[W + u]) + sum[2 * W + u]) + sum[3 * W + u];
      const int i = u / (16 * CT), col = col0 + u % (16 * CT);
      if (m0 + i < a.m && col < a.d) st1<DQ>(a.out, (part * a.m + m0 + i) * a.d + col, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t at = m0 + 16 * i + 4 * g + e;
          const int col = col0 + 16 * c + r;
          if (at < a.m && col < a.d) st1<DQ>(a.out, (part * a.m + at) * a.d + col, acc[i][c][e]);
        }
  }
}

// dq = the parts' sum, in an order that their number alone decides: one after
// the other, or 16 interleaved chains added in turn where there are many
template <int DQ>
__global__ __launch_bounds__(256) void k_cat_dq_sum_few(const float* part, int parts, int64_t values, void* out) {
  using namespace b8;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= values) return;
  if (i + 4 <= values && values % 4 == 0) {
    f32x4 v = *reinterpret_cast<const f32x4*>(part + i);
#pragma unroll 4
    for (int s = 1; s < parts; ++s) v += *reinterpret_cast<const f32x4*>(part + s * values + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) st1<DQ>(out, i + e, v[e]);
  } else {
    for (int64_t k = i; k < min(i + 4, values); ++k) {
      float v = part[k];
      for (int s = 1; s < parts; ++s) v += part[s * values + k];
      st1<DQ>(out, k, v);
    }
  }
}
template <int DQ>
__global__ __launch_bounds__(256) void k_cat_dq_sum(const float* part, int parts, int64_t values, void* out) {
  using namespace b8;
  __shared__ float chain[16][16];
  const int e = (int)threadIdx.x & 15, c = (int)threadIdx.x >> 4;
  const int64_t i = (int64_t)blockIdx.x * 16 + e;
  float v = 0.f;
  if (i < values) {
#pragma unroll 8
    for (int s = c; s < parts; s += 16) v += part[s * values + i];
  }
  chain[c][e] = v;
  __syncthreads();
  if (c == 0 && i < values) {
#pragma unroll
    for (int q = 1; q < 16; ++q) v += chain[q][e];
    st1<DQ>(out, i, v);
  }
}

}  // namespace tt
