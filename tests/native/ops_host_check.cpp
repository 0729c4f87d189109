// Host-side checks of the multi-tensor AdamW and 8-bit catalogue entries under
// AddressSanitizer.  Built by `make -C ceo-recommender_amd/csrc asan_ops` with
// their translation unit instrumented on the host side only; run on a CPU:
// calls that pass the checks reach launches that fail without a GPU, which is
// all right here.  Prints "ops_host_check: ALL OK" on success.
#include <cstdio>
#include <cstring>
#include <vector>

#include "../../include/ceo_tt.h"

static int failures = 0;
#define CHECK(cond)                                                          \
  do {                                                                       \
    if (!(cond)) {                                                           \
      std::fprintf(stderr, "FAILED %s:%d  %s\n", __FILE__, __LINE__, #cond); \
      ++failures;                                                            \
    }                                                                        \
  } while (0)

int main() {
  std::vector<float> buf(1 << 16);
  float* p = buf.data();
  uint8_t* b = reinterpret_cast<uint8_t*>(p);
  tt_adamw_state st;
  std::memset(&st, 0, sizeof(st));
  st.exp_avg = st.exp_avg_sq = p;
  st.m_codes = st.m_scales = st.r_codes = st.r_scales = b;
  st.n_blocks = 1 << 20;
  tt_adamw_hp hp = {1e-3, 0.9, 0.999, 1e-8, 0.01};
  // lists shorter and longer than a launch takes, empty tensors among them: the argument lists stay in bounds
  for (int n_t : {0, 1, 63, 64, 65, 128, 300}) {
    std::vector<tt_adamw_tensor> ts(n_t);
    for (int i = 0; i < n_t; ++i) ts[i] = tt_adamw_tensor{p, p, (int64_t)(i % 7 == 3 ? 0 : 1 + 37 * i), (int64_t)i * 100, 1 + i % 5, i % 3};
    for (int bits : {8, 32}) (void)tt_adamw_step(ts.data(), n_t, bits, &st, &hp, 1, nullptr);
    st.steps = reinterpret_cast<int64_t*>(p);
    st.coefs = p;
    st.n_steps = 1000;
    (void)tt_adamw_step(ts.data(), n_t, 8, &st, &hp, 1, nullptr);
    st.steps = nullptr;
  }
  tt_adamw_tensor t = {p, p, (int64_t)1 << 40, 0, 1, 0};
  CHECK(tt_adamw_step(&t, 1, 32, &st, &hp, 0, nullptr) == TT_ERR_ARG);  // more values than blocks
  CHECK(tt_adamw_step(nullptr, 1, 32, &st, &hp, 0, nullptr) == TT_ERR_ARG);
  CHECK(tt_adamw_step(&t, 1, 16, &st, &hp, 0, nullptr) == TT_ERR_UNSUPPORTED);
  CHECK(tt_adamw_held(&st, nullptr, p, nullptr) == TT_ERR_ARG);
  for (int64_t m : {1, 2, 16, 17, 64, 65, 1000, 16384, 1000000})
    for (int64_t n : {1, 100, 32771, 1000003})
      for (int32_t d : {1, 60, 128, 129, 512, 8192}) {
        CHECK(tt_cat_scores_workspace_bytes(m, n, d) >= 0);
        CHECK(tt_cat_dq_workspace_bytes(m, n, d, 0) >= 0);
        CHECK(tt_cat_dq_workspace_bytes(m, n, d, 1) >= 0);
        (void)tt_cat_scores(p, 0, m, d, d, b, b, n, p, 1, p, (int64_t)1 << 60, nullptr);
        (void)tt_cat_dq(p, 1, m, n, n, b, b, d, p, 1, p, (int64_t)1 << 60, nullptr);
      }
  CHECK(tt_cat_write(p, 0, 5, 8, 8, nullptr, 0, b, b, 4, nullptr, nullptr) == TT_ERR_ARG);
  CHECK(tt_cat_read(b, b, 4, 8, nullptr, 1, 4, p, 0, 8, nullptr) == TT_ERR_ARG);
  CHECK(tt_cat_scores_workspace_bytes(-1, 1, 1) == TT_ERR_ARG);
  CHECK(tt_cat_dq_workspace_bytes(1, 1, 0, 0) == TT_ERR_ARG);
  if (failures) {
    std::fprintf(stderr, "ops_host_check: %d FAILED\n", failures);
    return 1;
  }
  std::printf("ops_host_check: ALL OK\n");
  return 0;
}
