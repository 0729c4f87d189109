// Host side of the operators beside the two-tower path (a translation unit of
// its own): argument checks and launches of the multi-tensor AdamW step and
// of the 8-bit embedding catalogue, behind the C-ABI of include/ceo_tt.h.
#include <algorithm>
#include <climits>
#include <cmath>
#include <memory>
#include <new>
#include <type_traits>

#include "tt_adamw.hip"
#include "tt_catalogue.hip"

namespace tt {

static int ops_launch_check() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TT_OK : (int)e;
}
// rows in x, CAT_UNIT blocks of them in y
static dim3 cat_grid(int64_t m, int nkb) {
  return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>((m + 15) / 16, 16384)), (unsigned)((nkb + CAT_UNIT - 1) / CAT_UNIT));
}
static bool dtype_ok(int64_t dt) { return dt == TT_F32 || dt == TT_BF16 || dt == TT_F16; }
static bool aligned(const void* p, uintptr_t to) { return (uintptr_t)p % to == 0; }
static uintptr_t size_of(int32_t dt) { return dt == TT_F32 ? 4 : 2; }
static unsigned grid_for(int64_t work, int64_t per_block, int64_t most) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((work + per_block - 1) / per_block, most));
}

// F(std::integral_constant) for an element type known at run time
template <typename F>
static void with_dtype(int32_t dt, F f) {
  if (dt == TT_F32)
    f(std::integral_constant<int, TT_F32>{});
  else if (dt == TT_BF16)
    f(std::integral_constant<int, TT_BF16>{});
  else
    f(std::integral_constant<int, TT_F16>{});
}

// Raises every counter that the list names, once each.  Rising indices (one a
// tensor) go out as they come, others are sorted first.
static int adamw_advance(const tt_adamw_tensor* tensors, int32_t n, const tt_adamw_state& st, const tt_adamw_hp& hp,
                         uint64_t seed, hipStream_t s) {
  AdamwCounters a{st.steps, (AdamwCoef*)st.coefs, hp.lr, hp.beta1, hp.beta2, seed, {}, 0};
  bool rising = true;
  int64_t last = -1;
  for (int32_t i = 0; i < n; ++i) {
    rising = rising && tensors[i].step > last;
    last = tensors[i].step;
  }
  std::unique_ptr<uint32_t[]> sorted;
  int32_t count = n;
  if (!rising) {
    sorted.reset(new (std::nothrow) uint32_t[n]);
    if (!sorted) return (int)hipErrorOutOfMemory;
    for (int32_t i = 0; i < n; ++i) sorted[i] = (uint32_t)tensors[i].step;
    std::sort(sorted.get(), sorted.get() + n);
    count = (int32_t)(std::unique(sorted.get(), sorted.get() + n) - sorted.get());
  }
  for (int32_t i = 0; i < count;) {
    for (a.n = 0; i < count && a.n < ADAMW_LIST; ++i) a.at[a.n++] = sorted ? sorted[i] : (uint32_t)tensors[i].step;
    hipLaunchKernelGGL(k_adamw_advance, dim3(1), dim3(ADAMW_LIST), 0, s, a);
  }
  return ops_launch_check();
}

}  // namespace tt

using namespace tt;

extern "C" {

int32_t tt_adamw_step(const tt_adamw_tensor* tensors, int32_t n_tensors, int32_t state_bits,
                      const tt_adamw_state* state, const tt_adamw_hp* hp, uint64_t seed, tt_stream_t stream) {
  if (!state || !hp || n_tensors < 0 || (n_tensors > 0 && !tensors)) return TT_ERR_ARG;
  if (state_bits != 8 && state_bits != 32) return TT_ERR_UNSUPPORTED;
  if (!(hp->beta1 >= 0.0 && hp->beta1 < 1.0 && hp->beta2 >= 0.0 && hp->beta2 < 1.0)) return TT_ERR_ARG;
  for (const double x : {hp->lr, hp->eps, hp->weight_decay})
    if (!(x >= 0.0) || !std::isfinite(x)) return TT_ERR_ARG;
  if (state->n_blocks < 0 || state->n_blocks > (int64_t)UINT32_MAX) return TT_ERR_ARG;  // the hash takes 32 bits
  if (state->steps && (!state->coefs || state->n_steps > (int64_t)UINT32_MAX)) return TT_ERR_ARG;
  int64_t values = 0;
  for (int32_t i = 0; i < n_tensors; ++i) {
    const tt_adamw_tensor& t = tensors[i];
    if (t.n < 0 || !dtype_ok(t.dtype)) return TT_ERR_ARG;
    if (state->steps && (t.step < 0 || t.step >= state->n_steps)) return TT_ERR_ARG;
    if (t.n == 0) continue;  // its counter still counts
    const uintptr_t es = size_of((int32_t)t.dtype);
    if (!t.param || !t.grad || !aligned(t.param, es) || !aligned(t.grad, es)) return TT_ERR_ARG;
    const int64_t nb = (t.n - 1) / TT_BLOCK + 1;
    if (t.block0 < 0 || nb > state->n_blocks || t.block0 > state->n_blocks - nb) return TT_ERR_ARG;
    if (!state->steps && t.step < 1) return TT_ERR_ARG;
    values += t.n;
  }
  if (values > 0 && (state_bits == 32 ? !state->exp_avg || !state->exp_avg_sq
                                      : !state->m_codes || !state->m_scales || !state->r_codes || !state->r_scales))
    return TT_ERR_ARG;
  if (!aligned(state->exp_avg, 4) || !aligned(state->exp_avg_sq, 4) || !aligned(state->steps, 8) || !aligned(state->coefs, 4))
    return TT_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  AdamwArgs a;
  a.from_grad = hp->beta1 < 0.5;
  a.w1 = (float)(a.from_grad ? -hp->beta1 : 1.0 - hp->beta1);
  a.b2 = (float)hp->beta2;
  a.c2 = (float)(1.0 - hp->beta2);
  a.eps = (float)hp->eps;
  a.decay = (float)(1.0 - hp->lr * hp->weight_decay);
  a.m = state->exp_avg;
  a.v = state->exp_avg_sq;
  a.mc = state->m_codes;
  a.ms = state->m_scales;
  a.rc = state->r_codes;
  a.rs = state->r_scales;
  a.coefs = state->steps ? (const AdamwCoef*)state->coefs : nullptr;
  if (state->steps)
    if (const int rc = adamw_advance(tensors, n_tensors, *state, *hp, seed, s)) return rc;
  if (values == 0) return TT_OK;
  // 8-bit states of many values: 4 rounds a workgroup spare three of four looks for its tensor (one / four rounds, us,
  // bf16: 1 M values 8.2 / 11.5, 4 M 14.7 / 15.6, 8 M 26.4 / 23.7, 96 M 267 / 215; fp32: 4 M 18.4 / 17.8, 16 M 47.6 /
  // 46.1; 32-bit states of 96 M 517 / 528)
  const int64_t chunk = ADAMW_STRIDE * (state_bits == 8 && values >= 1 << 22 ? 4 : 1);
  int64_t last_step = 0;
  AdamwCoef last{};
  for (int32_t from = 0; from < n_tensors;) {
    int64_t chunks = 0;
    a.n_t = 0;
    for (; from < n_tensors && a.n_t < ADAMW_LIST; ++from) {
      const tt_adamw_tensor& t = tensors[from];
      if (t.n == 0) continue;
      const int64_t c = (t.n + chunk - 1) / chunk;
      if (c > INT32_MAX / 2) return TT_ERR_UNSUPPORTED;
      if (chunks + c > INT32_MAX / 2) break;
      const int k = a.n_t++;
      a.p[k] = t.param;
      a.g[k] = t.grad;
      a.n[k] = t.n;
      a.blk[k] = t.block0;
      a.dtype[k] = (uint8_t)t.dtype;
      a.first[k] = (int32_t)chunks;
      if (state->steps) {
        a.c[k] = AdamwCoef{0.f, 0.f, (uint32_t)t.step, 0u};
      } else {
        if (t.step != last_step) last = adamw_coef(hp->lr, hp->beta1, hp->beta2, seed, last_step = t.step);
        a.c[k] = last;
      }
      chunks += c;
    }
    if (a.n_t == 0) break;
    for (int k = a.n_t; k < ADAMW_LIST; ++k) a.first[k] = INT32_MAX;
    a.chunk = (int32_t)chunk;
    if (state_bits == 32)
      hipLaunchKernelGGL(k_adamw<32>, dim3((unsigned)chunks), dim3(ADAMW_THREADS), 0, s, a);
    else
      hipLaunchKernelGGL(k_adamw<8>, dim3((unsigned)chunks), dim3(ADAMW_THREADS), 0, s, a);
    if (const int rc = ops_launch_check()) return rc;
  }
  return TT_OK;
}

int32_t tt_adamw_held(const tt_adamw_state* state, void* m, void* r, tt_stream_t stream) {
  if (!state || state->n_blocks < 0) return TT_ERR_ARG;
  if (state->n_blocks == 0) return TT_OK;
  if (!state->m_codes || !state->m_scales || !state->r_codes || !state->r_scales || !m || !r) return TT_ERR_ARG;
  if (!aligned(m, 2) || !aligned(r, 2)) return TT_ERR_ARG;
  const int64_t n8 = state->n_blocks * b8::LANES;
  hipLaunchKernelGGL(k_adamw_held, dim3(grid_for(n8, 256, 8192), 2), dim3(256), 0, (hipStream_t)stream, state->m_codes,
                     state->m_scales, state->r_codes, state->r_scales, m, r, n8);
  return ops_launch_check();
}

// shared checks of the catalogue calls: sizes whose products stay in 63 bits
static bool cat_sizes_ok(int64_t rows, int32_t d) { return rows >= 0 && rows <= ((int64_t)1 << 40) && d >= 1 && d <= (1 << 20); }
static int cat_blocks(int32_t d) { return (d + TT_BLOCK - 1) / TT_BLOCK; }

int32_t tt_cat_write(const void* x, int32_t dtype, int64_t m, int64_t ldx, int32_t d, const int64_t* rows, int64_t row0,
                     uint8_t* codes, uint8_t* scales, int64_t capacity, int32_t* owner, tt_stream_t stream) {
  if (!cat_sizes_ok(m, d) || !cat_sizes_ok(capacity, d) || !dtype_ok(dtype) || (m > 1 && ldx < d)) return TT_ERR_ARG;
  if (rows && m >= INT32_MAX) return TT_ERR_ARG;  // a row's owner is a place in 31 bits
  if (!rows && (row0 < 0 || row0 > capacity - m)) return TT_ERR_ARG;
  if (m == 0 || capacity == 0) return TT_OK;
  if (rows && !owner) return TT_ERR_ARG;
  if (!x || !codes || !scales || !aligned(x, size_of(dtype)) || !aligned(rows, 8) || !aligned(owner, 4)) return TT_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const CatRows r{rows, row0, capacity};
  const int nkb = cat_blocks(d);
  if (rows && m <= CAT_FEW) {
    with_dtype(dtype, [&](auto t) {
      hipLaunchKernelGGL(k_cat_write_few<decltype(t)::value>, dim3(grid_for(m * nkb, 16, INT32_MAX)), dim3(256), 0, s, x,
                         (int)m, ldx, d, nkb, r, codes, scales);
    });
    return ops_launch_check();
  }
  if (rows) hipLaunchKernelGGL(k_cat_own, dim3(grid_for(m, 256, 4096)), dim3(256), 0, s, r, m, owner);
  with_dtype(dtype, [&](auto t) {
    hipLaunchKernelGGL(k_cat_write<decltype(t)::value>, cat_grid(m, nkb), dim3(256), 0, s, x, m, ldx,
                       d, nkb, r, codes, scales, rows ? owner : nullptr);
  });
  if (rows) hipLaunchKernelGGL(k_cat_disown, dim3(grid_for(m, 256, 4096)), dim3(256), 0, s, r, m, owner);
  return ops_launch_check();
}

int32_t tt_cat_read(const uint8_t* codes, const uint8_t* scales, int64_t capacity, int32_t d, const int64_t* rows,
                    int64_t row0, int64_t m, void* out, int32_t dtype, int64_t ldo, tt_stream_t stream) {
  if (!cat_sizes_ok(m, d) || !cat_sizes_ok(capacity, d) || !dtype_ok(dtype) || (m > 1 && ldo < d)) return TT_ERR_ARG;
  if (!rows && (row0 < 0 || row0 > capacity - m)) return TT_ERR_ARG;
  if (m == 0) return TT_OK;
  if (!out || (capacity > 0 && (!codes || !scales)) || !aligned(out, size_of(dtype)) || !aligned(rows, 8)) return TT_ERR_ARG;
  const CatRows r{rows, row0, capacity};
  const int nkb = cat_blocks(d);
  with_dtype(dtype, [&](auto t) {
    hipLaunchKernelGGL(k_cat_read<decltype(t)::value>, cat_grid(m, nkb), dim3(256), 0,
                       (hipStream_t)stream, codes, scales, r, m, d, nkb, out, ldo);
  });
  return ops_launch_check();
}

// Queries that each streaming workgroup encodes itself, at most 64 blocks in four
// rounds: no workspace, one launch.  Against a launch for the codes, us: 20 x 2000 x
// 128 4.6 / 6.4, 64 x 100000 x 128 10.8 / 12.3 (32-bit results 12.3 / 13.8), 37 x
// 1000003 x 128 42.1 / 45.1, 1 x 100000 x 256 7.3 / 9.6, 16 x 50000 x 512 10.7 / 13.4,
// 21 x 50000 x 384 11.3 / 11.1, 32 x 100000 x 256 12.0 / 15.2 (bf16).  More than 64
// blocks were not timed.
static bool cat_encodes(int64_t m, int nkb) { return m * nkb <= 64 && nkb <= 4; }

int64_t tt_cat_scores_workspace_bytes(int64_t m, int64_t n, int32_t d) {
  if (!cat_sizes_ok(m, d) || !cat_sizes_ok(n, d)) return TT_ERR_ARG;
  const int64_t nkb = cat_blocks(d);
  if (cat_encodes(m, (int)nkb)) return 0;
  return m * nkb * TT_BLOCK + (m * nkb + 255) / 256 * 256;  // codes | scales
}

}  // extern "C"

namespace tt {
template <int DT, int IT, int QT, int NKB>
static void launch_stream(StreamArgs& a, hipStream_t s) {
  const int64_t groups = (a.n + 64 * IT - 1) / (64 * IT);
  // two workgroups a CU; up to four of the form with the fewest registers, where each has four groups to walk over
  // (512 / 1024 / 2048 workgroups, us, bf16: 1 x 1000003 x 128 28.8 / 22.6 / 25.9, 1 x 300000 x 128 12.0 / 9.5 / 10.8, 8 x
  // 1000003 x 60 25.3 / 23.8 / 28.0, 16 x 1000003 x 128 26.8 / 29.0 / 30.9; other forms: 1 x 300000 x 256 15.9 / 17.1 /
  // 18.7, 16 x 300000 x 512 30.9 / 37.7 / 41.0, 32 x 1000003 x 128 36.1 / 39.4 / 40.0, 37 x 1000003 x 128 42.6 / 42.9 /
  // 47.9)
  const int64_t want = QT == 1 && NKB == 1 ? std::max<int64_t>(512, std::min<int64_t>(1024, groups / 4)) : 512;
  a.strips = std::min(groups, want);
  a.per = (a.strips + 7) / 8;
  hipLaunchKernelGGL((k_cat_stream<DT, IT, QT, NKB>), dim3((unsigned)(8 * a.per)), dim3(256), 0, s, a);
}
template <int DT>
static int launch_scores(StreamArgs& a, hipStream_t s) {
  if (a.m <= 64 && cat_encodes(a.m, a.nkb)) {  // at most 4 blocks a query, 3 of more than 16, 1 of more than 32
    auto* const f = a.m > 32     ? launch_stream<DT, 4, 4, 1>
                    : a.m > 16   ? a.nkb == 1   ? launch_stream<DT, 2, 2, 1>
                                   : a.nkb == 2 ? launch_stream<DT, 2, 2, 2>
                                                : launch_stream<DT, 2, 2, 3>
                    : a.nkb == 1 ? launch_stream<DT, 1, 1, 1>
                    : a.nkb == 2 ? launch_stream<DT, 1, 1, 2>
                    : a.nkb == 3 ? launch_stream<DT, 1, 1, 3>
                                 : launch_stream<DT, 1, 1, 4>;
    f(a, s);
    return TT_OK;
  }
  if (a.m <= 64) {
    // codes from the workspace are read again for every tile: kept in registers, 24 x 100000 x 384 took 18.4 us for
    // 17.3, 30 x 100000 x 512 21.6 for 21.7, and 64 x 100000 x 256 went to scratch (35 for 18)
    auto* const f = a.m > 32 ? launch_stream<DT, 4, 4, 0> : a.m > 16 ? launch_stream<DT, 2, 2, 0> : launch_stream<DT, 1, 1, 0>;
    f(a, s);
    return TT_OK;
  }
  const int64_t nt = (a.n + CT_N - 1) / CT_N, mt = (a.m + CT_M - 1) / CT_M;
  if (mt > INT32_MAX / 8 / nt) return TT_ERR_UNSUPPORTED;
  const int64_t per = (mt * nt + 7) / 8;
  hipLaunchKernelGGL(k_cat_scores<DT>, dim3((unsigned)(8 * per)), dim3(256), 0, s, (const uint8_t*)a.q, a.qs, a.m,
                     a.codes, a.scales, a.n, a.nkb, a.out, mt, nt, per, std::max(4, 32 / a.nkb));
  return TT_OK;
}
}  // namespace tt

extern "C" {

int32_t tt_cat_scores(const void* q, int32_t dtype, int64_t m, int64_t ldq, int32_t d, const uint8_t* codes,
                      const uint8_t* scales, int64_t n, void* out, int32_t out_dtype, void* ws, int64_t ws_bytes,
                      tt_stream_t stream) {
  if (!cat_sizes_ok(m, d) || !cat_sizes_ok(n, d) || !dtype_ok(dtype) || !dtype_ok(out_dtype) || (m > 1 && ldq < d))
    return TT_ERR_ARG;
  if (m == 0 || n == 0) return TT_OK;
  const int64_t need = tt_cat_scores_workspace_bytes(m, n, d);
  if (!q || !codes || !scales || !out || (need > 0 && !ws)) return TT_ERR_ARG;
  if (!aligned(q, size_of(dtype)) || !aligned(out, size_of(out_dtype)) || !aligned(codes, 16) || !aligned(ws, 16)) return TT_ERR_ARG;
  if (ws_bytes < need) return TT_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  StreamArgs a{};
  a.q = q;
  a.codes = codes;
  a.scales = scales;
  a.out = out;
  a.m = m;
  a.n = n;
  a.ldq = ldq;
  a.d = d;
  a.nkb = cat_blocks(d);
  a.q_dtype = dtype;
  if (need > 0) {
    uint8_t* qc = (uint8_t*)ws;
    uint8_t* qs = qc + m * a.nkb * TT_BLOCK;
    const CatRows r{nullptr, 0, m};
    with_dtype(dtype, [&](auto t) {
      hipLaunchKernelGGL(k_cat_write<decltype(t)::value>, cat_grid(m, a.nkb), dim3(256), 0, s, q, m,
                         ldq, d, a.nkb, r, qc, qs, (int32_t*)nullptr);
    });
    a.q = qc;
    a.qs = qs;
  }
  int rc = TT_OK;
  with_dtype(out_dtype, [&](auto t) { rc = launch_scores<decltype(t)::value>(a, s); });
  return rc ? rc : ops_launch_check();
}

}  // extern "C"

namespace tt {
// How dq's rows, columns and sum are split.  Parts of the catalogue until about
// two workgroups a CU have work, none shorter than 2 steps; a part writes m d
// floats and reads its share of the codes and of dS.  256 / 512 / 1024 workgroups,
// in us: 16384 x 32768 x 128 in bf16 326 / 229 / 277, 8192 x 100000 x 256 850 / 536 /
// 562, 1 x 1000003 x 128 28 / 27 / 31, 64 x 100000 x 256 21 / 25 / 32; 513 x 20011 x
// 512 in fp32 64 / 64 / 63.
struct DqPlan {
  int ct, rt, wm, groups;
  int64_t mt, splits, part_steps;
};
static DqPlan dq_plan(int64_t m, int64_t n, int32_t d, int32_t dtype) {
  DqPlan p;
  p.ct = d <= 64 ? 4 : d <= 128 ? 8 : 16;
  p.wm = m <= 16 ? 1 : 4;
  // two row tiles a wave where 16 columns of them leave room: with dS in two or three planes they go to scratch (8192 x
  // 100000 x 256 in fp16 1155 us for 902, 1000 x 20000 x 256 62 for 42; in bf16 541 for 649 with one)
  p.rt = m <= 64 || (dtype != TT_BF16 && p.ct == 16) ? 1 : 2;
  p.groups = (d + 16 * p.ct - 1) / (16 * p.ct);
  p.mt = (m + 16 * p.rt * p.wm - 1) / (16 * p.rt * p.wm);
  const int64_t step = p.wm == 1 ? 128 : 64, steps = std::max<int64_t>(1, (n + step - 1) / step);
  const int64_t blocks = p.mt * p.groups;
  int64_t s = std::max<int64_t>(1, std::min<int64_t>((512 + blocks - 1) / blocks, steps / 2));
  p.part_steps = (steps + s - 1) / s;
  p.splits = (steps + p.part_steps - 1) / p.part_steps;
  return p;
}

template <int DT, int DQ, int CT, int RT, int WM, bool ODD>
static void launch_dq_as(const DqArgs& a, hipStream_t s) {
  constexpr int LDS = dq_lds<CT, WM>();
  if constexpr (LDS > 64 * 1024)  // (every time: it holds for the current device)
    (void)hipFuncSetAttribute((const void*)k_cat_dq<DT, DQ, CT, RT, WM, ODD>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  hipLaunchKernelGGL((k_cat_dq<DT, DQ, CT, RT, WM, ODD>), dim3((unsigned)(8 * a.per)), dim3(256), LDS, s, a);
}
template <int DT, int DQ, int CT, int RT, int WM>
static void launch_dq_one(const DqArgs& a, hipStream_t s) {
  // 16 columns of two row tiles have no registers for the fifth word (scratch: 8192 x 100001 x 256 832 us for 752)
  if constexpr (DT != TT_F32 && !(CT == 16 && RT == 2)) {
    if (a.lds % 2 && (uintptr_t)a.ds % 4 == 0 && a.m > 1) return launch_dq_as<DT, DQ, CT, RT, WM, true>(a, s);
  }
  launch_dq_as<DT, DQ, CT, RT, WM, false>(a, s);
}
template <int DT, int DQ, int CT>
static void launch_dq_rows(const DqArgs& a, const DqPlan& p, hipStream_t s) {
  if (p.wm == 1)
    launch_dq_one<DT, DQ, CT, 1, 1>(a, s);
  else if (p.rt == 1)
    launch_dq_one<DT, DQ, CT, 1, 4>(a, s);
  else if constexpr (DT == TT_BF16 || CT < 16)
    launch_dq_one<DT, DQ, CT, 2, 4>(a, s);
}
template <int DT, int DQ>
static void launch_dq(const DqArgs& a, const DqPlan& p, hipStream_t s) {
  if (p.ct == 4)
    launch_dq_rows<DT, DQ, 4>(a, p, s);
  else if (p.ct == 8)
    launch_dq_rows<DT, DQ, 8>(a, p, s);
  else
    launch_dq_rows<DT, DQ, 16>(a, p, s);
}
}  // namespace tt

extern "C" {

int64_t tt_cat_dq_workspace_bytes(int64_t m, int64_t n, int32_t d, int32_t ds_dtype) {
  if (!cat_sizes_ok(m, d) || !cat_sizes_ok(n, d) || !dtype_ok(ds_dtype)) return TT_ERR_ARG;
  if (m == 0) return 0;
  const DqPlan p = dq_plan(m, n, d, ds_dtype);
  return p.splits > 1 ? p.splits * m * d * (int64_t)sizeof(float) : 0;
}

int32_t tt_cat_dq(const void* ds, int32_t ds_dtype, int64_t m, int64_t lds, int64_t n, const uint8_t* codes,
                  const uint8_t* scales, int32_t d, void* dq, int32_t dq_dtype, void* ws, int64_t ws_bytes,
                  tt_stream_t stream) {
  if (!cat_sizes_ok(m, d) || !cat_sizes_ok(n, d) || !dtype_ok(ds_dtype) || !dtype_ok(dq_dtype) || (m > 1 && lds < n))
    return TT_ERR_ARG;
  if (m == 0) return TT_OK;
  if (!dq || (n > 0 && (!ds || !codes || !scales))) return TT_ERR_ARG;
  const int64_t need = tt_cat_dq_workspace_bytes(m, n, d, ds_dtype);
  if (need > 0 && (!ws || ws_bytes < need)) return TT_ERR_WORKSPACE;
  if (!aligned(ds, size_of(ds_dtype)) || !aligned(dq, size_of(dq_dtype)) || !aligned(codes, 16) || !aligned(ws, 16)) return TT_ERR_ARG;
  const DqPlan p = dq_plan(m, n, d, ds_dtype);
  if (p.mt > INT32_MAX / 16 / p.groups / p.splits) return TT_ERR_UNSUPPORTED;
  hipStream_t s = (hipStream_t)stream;
  DqArgs a;
  a.ds = ds;
  a.m = m;
  a.lds = lds;
  a.n = n;
  a.codes = codes;
  a.scales = scales;
  a.d = d;
  a.nkb = cat_blocks(d);
  a.out = p.splits > 1 ? ws : dq;
  a.mt = p.mt;
  a.splits = p.splits;
  a.per = (p.mt * p.groups * p.splits + 7) / 8;
  a.groups = p.groups;
  a.part_steps = p.part_steps;
  with_dtype(ds_dtype, [&](auto t) {
    constexpr int DT = decltype(t)::value;
    if (p.splits > 1)
      launch_dq<DT, TT_F32>(a, p, s);
    else
      with_dtype(dq_dtype, [&](auto u) { launch_dq<DT, decltype(u)::value>(a, p, s); });
  });
  if (p.splits > 1) {
    const int64_t values = m * d;
    const bool few = p.splits <= 16;
    const int64_t blocks = few ? (values + 1023) / 1024 : (values + 15) / 16;
    if (blocks > INT32_MAX) return TT_ERR_UNSUPPORTED;
    with_dtype(dq_dtype, [&](auto u) {
      if (few)
        hipLaunchKernelGGL(k_cat_dq_sum_few<decltype(u)::value>, dim3((unsigned)blocks), dim3(256), 0, s,
                           (const float*)ws, (int)p.splits, values, dq);
      else
        hipLaunchKernelGGL(k_cat_dq_sum<decltype(u)::value>, dim3((unsigned)blocks), dim3(256), 0, s, (const float*)ws,
                           (int)p.splits, values, dq);
    });
  }
  return ops_launch_check();
}

}  // extern "C"
