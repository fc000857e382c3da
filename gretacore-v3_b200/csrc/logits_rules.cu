// Rules on logits (penalties for repeated tokens, biases, a grammar's mask) and the arg-max of what they leave, in one pass.
//
// Bytes are what bounds it: logits in and out once, the mask's bits once.  A row belongs to a cluster of CTAs, a slice of the vocabulary to each; a CTA
// counts the history's ids that fall into its slice in shared memory (integer atomics: the counts do not depend on their order), so there is no table
// of counts to keep per sequence, to clear or to roll back, and a token that occurs often is adjusted once.  The history is read by every CTA of the
// row, from L2.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "greta_common.cuh"

using namespace greta;

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t LR_THREADS = 1024, LR_SLICE = 24576;  // tokens whose counts (and biases) a CTA holds at a time: 96 KB each
constexpr uint32_t LR_SEEN = 0x80000000u;

struct LogitsArgs {
  greta_logits_rules r;
  const void *in;
  void *out;
  uint32_t ld, ld_out, V, slice;
  int32_t *next;
  uint32_t *pos;
  bool vec, advance;
};

template <int FMT>
struct Elem;
template <>
struct Elem<GRETA_FMT_F32> {
  typedef float T;
  static __device__ __forceinline__ float load(T x) { return x; }
  static __device__ __forceinline__ T store(float x) { return x; }
};
template <>
struct Elem<GRETA_FMT_F16> {
  typedef __half T;
  static __device__ __forceinline__ float load(T x) { return __half2float(x); }
  static __device__ __forceinline__ T store(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<GRETA_FMT_BF16> {
  typedef __nv_bfloat16 T;
  static __device__ __forceinline__ float load(T x) { return __bfloat162float(x); }
  static __device__ __forceinline__ T store(float x) { return __float2bfloat16_rn(x); }
};

__device__ __forceinline__ bool better(float v, uint32_t i, float bv, uint32_t bi) { return v > bv || (v == bv && i < bi); }
__device__ __forceinline__ void warp_first_max(float &best, uint32_t &bi) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, best, o);
    const uint32_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
    if (better(ov, oi, best, bi)) {
      best = ov;
      bi = oi;
    }
  }
}

template <int FMT>
__global__ void __launch_bounds__(LR_THREADS) logits_rules_kernel(const __grid_constant__ LogitsArgs a) {
  typedef typename Elem<FMT>::T T;
  extern __shared__ uint32_t table[];  // [slice] counts of generated ids, LR_SEEN for any; behind them [slice] 1 + index of the last bias
  __shared__ float sv[32];
  __shared__ uint32_t si[32];
  cg::cluster_group cluster = cg::this_cluster();
  pdl_launch_dependents();
  pdl_wait();
  const greta_logits_rules &r = a.r;
  const uint32_t m = blockIdx.y, rank = blockIdx.x, ctas = gridDim.x, tid = threadIdx.x;
  const uint32_t per = (((a.V + ctas - 1) / ctas) + 31) & ~31u;  // slices of whole mask words
  const uint32_t lo = min(a.V, rank * per), hi = min(a.V, lo + per);
  const bool counts = r.ids && (r.repetition || r.frequency || r.presence);
  const uint32_t n_ids = r.ids ? min(r.n_ids[m], r.ld_ids) : 0;
  const uint32_t n_prompt = r.n_prompt ? r.n_prompt[m] : 0;
  const int32_t *ids = r.ids + (size_t)m * r.ld_ids;
  const float rep = r.ids && r.repetition ? r.repetition[m] : 1.f, freq = r.ids && r.frequency ? r.frequency[m] : 0.f,
              pres = r.ids && r.presence ? r.presence[m] : 0.f;
  const uint32_t b0 = r.bias_ids ? r.bias_start[m] : 0, b1 = r.bias_ids ? r.bias_start[m + 1] : 0;
  const uint32_t *allowed = r.allowed ? r.allowed + (size_t)m * r.ld_allowed : nullptr;
  const T *in = static_cast<const T *>(a.in) + (size_t)m * a.ld;
  T *out = a.out ? static_cast<T *>(a.out) + (size_t)m * a.ld_out : nullptr;
  uint32_t *biases = table + a.slice;

  float best = -INFINITY;
  uint32_t bi = 0xffffffffu;
  for (uint32_t c0 = lo; c0 < hi; c0 += a.slice) {
    const uint32_t n = min(a.slice, hi - c0);
    if (counts || r.bias_ids) {
      __syncthreads();
      if (counts)
        for (uint32_t i = tid; i < n; i += LR_THREADS) table[i] = 0;
      if (r.bias_ids)
        for (uint32_t i = tid; i < n; i += LR_THREADS) biases[i] = 0;
      __syncthreads();
      if (counts) {
#pragma unroll 4
        for (uint32_t i = tid; i < n_ids; i += LR_THREADS) {
          const uint32_t t = (uint32_t)ids[i] - c0;
          if (t < n) {
            if (i < n_prompt)
              atomicOr(&table[t], LR_SEEN);
            else
              atomicAdd(&table[t], 1u);
          }
        }
      }
      for (uint32_t i = b0 + tid; i < b1; i += LR_THREADS) {
        const uint32_t t = (uint32_t)r.bias_ids[i] - c0;
        if (t < n) atomicMax(&biases[t], i - b0 + 1);
      }
      __syncthreads();
    }
    // Every operation rounds once, in the order of the rules: no product is folded into the sum behind it.
    auto rule = [&](float x, uint32_t t, uint32_t word) {
      if (counts) {
        const uint32_t c = table[t - c0];
        if (c) {
          x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
          const uint32_t k = c & ~LR_SEEN;
          if (k) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)k)), pres);
        }
      }
      if (r.bias_ids) {
        const uint32_t b = biases[t - c0];
        if (b) x = __fadd_rn(x, r.bias[b0 + b - 1]);
      }
      if (!(word >> (t & 31) & 1)) x = -INFINITY;
      return Elem<FMT>::store(x);
    };
    auto look = [&](T y, uint32_t t) {
      float v = Elem<FMT>::load(y);
      if (v != v) v = t ? -INFINITY : INFINITY;  // as greta_cuda_argmax
      if (v > best || bi == 0xffffffffu) {       // a thread's tokens ascend
        best = v;
        bi = t;
      }
    };
    if (a.vec) {
      constexpr uint32_t W = 16 / sizeof(T);  // tokens of 16 bytes; c0 is a multiple of 32
      struct alignas(16) Pack { T x[W]; };
      const uint32_t whole = n / W;
#pragma unroll 2
      for (uint32_t i = tid; i < whole; i += LR_THREADS) {
        const uint32_t t = c0 + i * W;
        Pack p = *reinterpret_cast<const Pack *>(in + t);
        const uint32_t word = allowed ? allowed[t / 32] : 0xffffffffu;
#pragma unroll
        for (uint32_t e = 0; e < W; ++e) p.x[e] = rule(Elem<FMT>::load(p.x[e]), t + e, word);
        if (out) *reinterpret_cast<Pack *>(out + t) = p;
#pragma unroll
        for (uint32_t e = 0; e < W; ++e) look(p.x[e], t + e);
      }
      const uint32_t t = c0 + whole * W + tid;
      if (t < c0 + n) {
        const T y = rule(Elem<FMT>::load(in[t]), t, allowed ? allowed[t / 32] : 0xffffffffu);
        if (out) out[t] = y;
        look(y, t);
      }
    } else {
#pragma unroll 2
      for (uint32_t t = c0 + tid; t < c0 + n; t += LR_THREADS) {
        const T y = rule(Elem<FMT>::load(in[t]), t, allowed ? allowed[t / 32] : 0xffffffffu);
        if (out) out[t] = y;
        look(y, t);
      }
    }
  }
  if (!a.next) return;
  warp_first_max(best, bi);
  const uint32_t w = tid >> 5, l = tid & 31;
  if (l == 0) {
    sv[w] = best;
    si[w] = bi;
  }
  __syncthreads();
  if (w == 0) {
    best = sv[l];
    bi = si[l];
    warp_first_max(best, bi);
    __syncwarp();
    if (l == 0) {
      sv[0] = best;
      si[0] = bi;
    }
  }
  if (ctas > 1) cluster.sync();  // behind every CTA's reading of the history, too
  if (w == 0 && rank == 0) {
    if (ctas > 1) {
      best = -INFINITY;
      bi = 0xffffffffu;
      if (l < ctas) {
        best = *cluster.map_shared_rank(&sv[0], l);
        bi = *cluster.map_shared_rank(&si[0], l);
      }
      warp_first_max(best, bi);
    }
    if (l == 0) {
      a.next[m] = (int32_t)bi;
      if (a.advance) {
        if (n_ids < r.ld_ids) {
          r.ids[(size_t)m * r.ld_ids + n_ids] = (int32_t)bi;
          r.n_ids[m] = n_ids + 1;
        }
        if (a.pos) a.pos[m] = a.pos[m] + 1;
      }
    }
  }
  if (ctas > 1) cluster.sync();  // a CTA's shared memory outlives rank 0's reads
}

template <int FMT>
int launch_rules(cudaStream_t stream, LogitsArgs &a, uint32_t M) {
  // As the arg-max: rows that one CTA covers with a few loads per thread stay with it.
  const unsigned ctas = a.V <= 4096 ? 1 : (a.V <= 8192 ? 2 : (a.V <= 16384 ? 4 : 8));
  const uint32_t per = (((a.V + ctas - 1) / ctas) + 31) & ~31u;
  a.slice = std::min(LR_SLICE, per);
  const bool counts = a.r.ids && (a.r.repetition || a.r.frequency || a.r.presence);
  const size_t smem = counts || a.r.bias_ids ? (size_t)a.slice * 4 * (a.r.bias_ids ? 2 : 1) : 0;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    GRETA_CUDA_TRY(cudaFuncSetAttribute(logits_rules_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(LR_SLICE * 8)));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  GRETA_CUDA_TRY(launch_pdl_cluster(logits_rules_kernel<FMT>, dim3(ctas, M), dim3(LR_THREADS), ctas, smem, stream, a));
  return launched("logits_rules_kernel");
}

int adjust(greta_stream_t stream, const greta_logits_rules *rules, int fmt, const void *logits, uint32_t ld, void *out, uint32_t ld_out, uint32_t M, uint32_t V,
           int32_t *d_next, uint32_t *d_pos, bool advance, const char *name) {
  GRETA_REQUIRE(fmt == GRETA_FMT_F32 || fmt == GRETA_FMT_F16 || fmt == GRETA_FMT_BF16, "%s: format %d is not fp32, fp16 or bf16", name, fmt);
  if (M == 0) return GRETA_OK;
  GRETA_REQUIRE(V > 0 && V < 0x7fffffffu && M <= 65535, "%s: %u rows of %u logits", name, M, V);
  GRETA_REQUIRE(rules && logits && (out || d_next), "%s: null pointer", name);
  GRETA_REQUIRE(ld >= V && (!out || ld_out >= V), "%s: rows of %u logits, %u and %u apart", name, V, ld, ld_out);
  GRETA_REQUIRE(out != logits || ld == ld_out, "%s: in place with rows %u and %u apart", name, ld, ld_out);
  GRETA_REQUIRE(!rules->ids || (rules->n_ids && rules->ld_ids), "%s: ids without their number", name);
  GRETA_REQUIRE(!rules->bias_ids || (rules->bias && rules->bias_start), "%s: bias_ids without bias or bias_start", name);
  GRETA_REQUIRE(!rules->allowed || rules->ld_allowed >= (V + 31) / 32, "%s: %u words of mask for %u logits", name, rules->ld_allowed, V);
  GRETA_REQUIRE(!advance || (d_next && rules->ids), "%s: nothing to append to", name);
  const uint32_t size = fmt == GRETA_FMT_F32 ? 4 : 2;
  GRETA_REQUIRE((uintptr_t)logits % size == 0 && (uintptr_t)out % size == 0, "%s: misaligned pointer", name);
  LogitsArgs a{};
  a.r = *rules;
  a.in = logits;
  a.out = out;
  a.ld = ld;
  a.ld_out = ld_out;
  a.V = V;
  a.next = d_next;
  a.pos = d_pos;
  a.advance = advance;
  a.vec = aligned16(logits) && aligned16(out) && (size_t)ld * size % 16 == 0 && (!out || (size_t)ld_out * size % 16 == 0);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return fmt == GRETA_FMT_F32 ? launch_rules<GRETA_FMT_F32>(s, a, M) : fmt == GRETA_FMT_F16 ? launch_rules<GRETA_FMT_F16>(s, a, M) : launch_rules<GRETA_FMT_BF16>(s, a, M);
}

}  // namespace

extern "C" {

int greta_cuda_logits_adjust(greta_stream_t stream, const greta_logits_rules *rules, int fmt, const void *logits, uint32_t ld, void *out, uint32_t ld_out,
                             uint32_t M, uint32_t V, int32_t *d_next) {
  return adjust(stream, rules, fmt, logits, ld, out, ld_out, M, V, d_next, nullptr, false, "logits_adjust");
}
int greta_cuda_logits_adjust_advance(greta_stream_t stream, const greta_logits_rules *rules, int fmt, const void *logits, uint32_t ld, void *out,
                                     uint32_t ld_out, uint32_t M, uint32_t V, int32_t *d_next, uint32_t *d_pos) {
  return adjust(stream, rules, fmt, logits, ld, out, ld_out, M, V, d_next, d_pos, true, "logits_adjust_advance");
}

}  // extern "C"
