// Arguments, workspace and the slow path that the two forms of the paged attention share.
#pragma once
#include <cuda.h>

#include "paged.cuh"

namespace greta {

int gemm_ts_error_word(int **word);  // gemm_ts.cu: the word that greta_cuda_gemm_segments_status reads

struct PagedAttnArgs {
  CUtensorMap k, v;  // the pools as rows of `dim` elements; rows outside read as zeros
  CUtensorMap qm;    // queries of 16 bits
  greta_paged_cache c;
  greta_ragged r;
  const void *q;
  void *o;
  uint32_t ld_q, ld_o, group, window;
  float scale2;      // scale * log2(e)
  uint32_t *tickets;  // [PAGED_MAX_CTAS], zero between calls
  float *parts;       // PAGED_PARTS floats
  int *error;         // where a wait that gave up is reported
};

constexpr uint32_t PAGED_CTAS_PER_SM = 2, PAGED_MAX_CTAS = 512;  // of the form for few rows
constexpr uint32_t PAGED_TC_CTAS = 192;                          // of the form for portions
constexpr uint32_t PAGED_TICKETS = 65536;                        // bytes
constexpr uint32_t PAGED_COUNTER = PAGED_TICKETS / 4 - 1;        // the word that blocks are drawn from
constexpr uint32_t PAGED_MMA_PART = 64 * (128 + 2), PAGED_PART = 256 * (128 + 2);  // floats of a part of a row block
constexpr size_t PAGED_PARTS = 2 * (size_t)(PAGED_MAX_CTAS * PAGED_MMA_PART > PAGED_TC_CTAS * PAGED_PART ? PAGED_MAX_CTAS * PAGED_MMA_PART : PAGED_TC_CTAS * PAGED_PART);

bool paged_tc_fits(const PagedAttnArgs &w);
int paged_attn_tc(cudaStream_t stream, PagedAttnArgs &w, uint32_t heads);  // paged_attention_tc.cu

#ifdef __CUDACC__
// Elements elem(0 .. N - 1) of row R's unnormalised output over the keys k0 .. k1 - 1 (all seen by the row), whose scores are taken against mx and weights are `gain` times as large: again, where the
// product with hidden keys' values left no finite numbers.  Where values that the row sees are none either, they decide: their sum.  Rare and slow: a key at a time, by one
// thread.  Inlined, and its arrays in local memory: around a call the caller's loops would keep their sums there.  Not for rows whose sum of weights is no finite number: their outputs are none whatever the values are.
template <int N, typename Elem>
__device__ __forceinline__ void paged_again(const PagedAttnArgs &w, bool bf16, bool f32, uint32_t b, const PagedSeq &s, uint32_t g, uint32_t R, Elem elem, int k0, int k1, float mx,
                                         float gain, float (&y)[N]) {
  const uint32_t d = w.c.dim;
  const int32_t *table = w.c.table + (size_t)b * w.c.ld_table;
  auto value = [&](const void *p, size_t i) {
    const uint16_t x = static_cast<const uint16_t *>(p)[i];
    return bf16 ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
  };
  uint32_t again = 0;
#pragma unroll 1
  for (int n = 0; n < N; ++n)
    if (elem(n) < d && !isfinite(y[n])) again |= 1u << n;
  auto row_of = [&](int j, size_t &row) {  // false: no page, values of zero
    const int id = table[(uint32_t)j / w.c.page];
    row = (((size_t)id * w.c.kv_heads + g) * w.c.page + (uint32_t)j % w.c.page) * d;
    return id >= 0 && (uint32_t)id < w.c.pages;
  };
  size_t row;
  float acc[N];
#pragma unroll 1
  for (int n = 0; n < N; ++n) acc[n] = 0.f;
  if (!again) return;
  for (int j = k0; j < k1; ++j) {
    if (!row_of(j, row)) continue;
#pragma unroll 1
    for (int n = 0; n < N; ++n)
      if (again >> n & 1) {
        const float x = value(w.c.v, row + elem(n));
        if (!isfinite(x)) acc[n] += x;
      }
  }
#pragma unroll 1
  for (int n = 0; n < N; ++n)
    if (again >> n & 1 && acc[n] != 0.f) {
      y[n] = acc[n];
      again &= ~(1u << n);
    }
  if (!again) return;
  const size_t qi = (size_t)(s.first + R / w.group) * w.ld_q + (size_t)(g * w.group + R % w.group) * d;
  for (int j = k0; j < k1; ++j) {
    if (!row_of(j, row)) continue;
    float t = 0.f;
#pragma unroll 2
    for (uint32_t i = 0; i < d; ++i) t = fmaf(f32 ? static_cast<const float *>(w.q)[qi + i] : value(w.q, qi + i), value(w.c.k, row + i), t);
    const float p = gain * exp2f(t * w.scale2 - mx);
#pragma unroll 1
    for (int n = 0; n < N; ++n)
      if (again >> n & 1) acc[n] = fmaf(p, value(w.c.v, row + elem(n)), acc[n]);
  }
#pragma unroll 1
  for (int n = 0; n < N; ++n)
    if (again >> n & 1) y[n] = acc[n];
}
#endif


}  // namespace greta
