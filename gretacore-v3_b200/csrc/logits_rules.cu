// Rules on logits (penalties for repeated tokens, biases, a grammar's mask) and the arg-max of what they leave, in one pass.
//
// Bytes are what bounds it: logits in and out once, the mask's bits once.  A row belongs to a cluster of CTAs, a slice of the vocabulary to each.  A CTA
// reads the history once and keeps what falls into its slice, then goes through the slice in chunks of 16 tokens a thread: counts of the chunk's ids in shared memory
// (integer atomics: they do not depend on their order), so there is no table of counts to keep per sequence, to clear or to roll back, and a token that
// occurs often is adjusted once.  The chunk's logits are asked for before its counts are made.  Clusters of CTAs as large as the rows leave
// room for.  64 rows of 128256 logits, 4096 ids, 300 biases, masks: 32 us (2.1 TB/s; with one chunk of the whole slice a CTA 59): the phases of a chunk wait for
// one another, a division and a bias for every token of the text are issued at a few lanes a warp.  One row of 32000, 700 ids: 5.8 us, launch and cluster barriers.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "greta_common.cuh"

using namespace greta;

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t LR_EACH = 16;   // tokens of a thread and chunk
constexpr uint32_t LR_IDS = 2048, LR_BIASES = 512;  // of a slice that are kept; with more of them every chunk reads the caller's again
constexpr uint32_t LR_SEEN = 0x80000000u;

struct LogitsArgs {
  greta_logits_rules r;
  const void *in;
  void *out;
  uint32_t ld, ld_out, V;
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
__global__ void __launch_bounds__(1024) logits_rules_kernel(const __grid_constant__ LogitsArgs a) {
  typedef typename Elem<FMT>::T T;
  constexpr uint32_t W = 16 / sizeof(T), PACKS = LR_EACH / W;  // tokens of 16 bytes, pieces of a thread and chunk
  struct alignas(16) Pack { T x[W]; };
  extern __shared__ uint4 smem4[];
  __shared__ float sv[32];
  __shared__ uint32_t si[32];
  __shared__ uint32_t kept[2], n_later;  // ids and biases of the slice
  cg::cluster_group cluster = cg::this_cluster();
  pdl_launch_dependents();
  pdl_wait();
  const greta_logits_rules &r = a.r;
  const uint32_t m = blockIdx.y, rank = blockIdx.x, ctas = gridDim.x, tid = threadIdx.x, lane = tid & 31, threads = blockDim.x, chunk = threads * LR_EACH;
  const uint32_t per = (((a.V + ctas - 1) / ctas) + 31) & ~31u;  // slices of whole mask words
  const uint32_t lo = min(a.V, rank * per), hi = min(a.V, lo + per);
  const bool counts = r.ids && (r.repetition || r.frequency || r.presence), biased = r.bias_ids;
  // [chunk] counts of generated ids, LR_SEEN for any; [chunk] 1 + index of the last bias; the slice's ids (LR_SEEN: of the prompt); its biases' tokens and indices
  uint32_t *table = reinterpret_cast<uint32_t *>(smem4), *biases = table + (counts ? chunk : 0);
  uint32_t *list = biases + (biased ? chunk : 0), *bias_at = list + (counts ? LR_IDS : 0), *bias_of = bias_at + (biased ? LR_BIASES : 0);
  uint16_t *later = reinterpret_cast<uint16_t *>(bias_of + (biased ? LR_BIASES : 0));  // [chunk] tokens that ids or biases are about
  const uint32_t n_ids = r.ids ? min(r.n_ids[m], r.ld_ids) : 0;
  const uint32_t n_prompt = r.n_prompt ? r.n_prompt[m] : 0;
  const int32_t *ids = r.ids + (size_t)m * r.ld_ids;
  const float rep = r.ids && r.repetition ? r.repetition[m] : 1.f, freq = r.ids && r.frequency ? r.frequency[m] : 0.f,
              pres = r.ids && r.presence ? r.presence[m] : 0.f;
  const uint32_t b0 = biased ? r.bias_start[m] : 0, b1 = biased ? r.bias_start[m + 1] : 0;
  const uint32_t *allowed = r.allowed ? r.allowed + (size_t)m * r.ld_allowed : nullptr;
  const T *in = static_cast<const T *>(a.in) + (size_t)m * a.ld;
  T *out = a.out ? static_cast<T *>(a.out) + (size_t)m * a.ld_out : nullptr;
  // What lies in tokens from .. from + n - 1: count(token - from, of the prompt), bias(token - from, index).
  auto each_id = [&](uint32_t from, uint32_t n, auto count) {
#pragma unroll 4
    for (uint32_t i = tid; i < n_ids; i += threads) {
      const uint32_t t = (uint32_t)ids[i] - from;
      if (t < n) count(t, i < n_prompt);
    }
  };
  auto each_bias = [&](uint32_t from, uint32_t n, auto bias) {
    for (uint32_t i = b0 + tid; i < b1; i += threads) {
      const uint32_t t = (uint32_t)r.bias_ids[i] - from;
      if (t < n) bias(t, i - b0 + 1);
    }
  };
  auto to_table = [&](uint32_t t, bool prompt) {
    if (prompt)
      atomicOr(&table[t], LR_SEEN);
    else
      atomicAdd(&table[t], 1u);
  };
  const bool listed = hi - lo > chunk;  // more chunks than one: the lists are read once
  // Clear to begin with; every entry is cleared again by the one who uses it.
  for (uint32_t i = tid; i < chunk / 4 * (counts + biased); i += threads) reinterpret_cast<uint4 *>(table)[i] = make_uint4(0, 0, 0, 0);
  if (tid < 2) kept[tid] = 0;
  if (tid == 0) n_later = 0;
  if (listed && (counts || biased)) {
    __syncthreads();
    if (counts)
      for (uint32_t i0 = tid & ~31u; i0 < n_ids; i0 += 4 * threads) {  // places are given out by warps: a thousand single ones take 3 us
        uint32_t t[4];
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x) {
          const uint32_t i = i0 + x * threads + lane;
          t[x] = i < n_ids ? (uint32_t)ids[i] - lo : 0xffffffffu;
        }
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x) {
          const uint32_t in_slice = __ballot_sync(0xffffffffu, t[x] < hi - lo);
          if (!in_slice) continue;
          uint32_t at = 0;
          if (lane == 0) at = atomicAdd(&kept[0], __popc(in_slice));
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(in_slice & ((1u << lane) - 1));
          if (t[x] < hi - lo && at < LR_IDS) list[at] = t[x] | (i0 + x * threads + lane < n_prompt ? LR_SEEN : 0);
        }
      }
    if (biased)
      each_bias(lo, hi - lo, [&](uint32_t t, uint32_t i) {
        const uint32_t x = atomicAdd(&kept[1], 1u);
        if (x < LR_BIASES) {
          bias_at[x] = t;
          bias_of[x] = i;
        }
      });
  }

  float best = -INFINITY;
  uint32_t bi = 0xffffffffu, above = 0;  // above: the largest that the warp has seen, as an ordered integer
  for (uint32_t c0 = lo; c0 < hi; c0 += chunk) {
    const uint32_t n = min(chunk, hi - c0), whole = a.vec ? n / W : 0;
    Pack p[PACKS];
    uint32_t word[PACKS];
#pragma unroll
    for (uint32_t k = 0; k < PACKS; ++k) {
      const uint32_t i = k * threads + tid;
      word[k] = 0xffffffffu;
      if (i < whole) {
        p[k] = *reinterpret_cast<const Pack *>(in + c0 + i * W);  // c0 is a multiple of 32
        if (allowed) word[k] = allowed[(c0 + i * W) / 32];
      }
    }
    if (counts || biased) {
      __syncthreads();  // the tables are clear, the lists are there
      if (counts) {
        if (listed && kept[0] <= LR_IDS) {
          for (uint32_t i = tid; i < kept[0]; i += threads) {
            const uint32_t t = (list[i] & ~LR_SEEN) + lo - c0;
            if (t < n) to_table(t, list[i] & LR_SEEN);
          }
        } else {
          each_id(c0, n, to_table);
        }
      }
      if (biased) {
        if (listed && kept[1] <= LR_BIASES) {
          for (uint32_t i = tid; i < kept[1]; i += threads) {
            const uint32_t t = bias_at[i] + lo - c0;
            if (t < n) atomicMax(&biases[t], bias_of[i]);
          }
        } else {
          each_bias(c0, n, [&](uint32_t t, uint32_t i) { atomicMax(&biases[t], i); });
        }
      }
      __syncthreads();
    }
    // Every operation rounds once, in the order of the rules: no product is folded into the sum behind it.
    auto rule = [&](float x, uint32_t t, uint32_t word, uint32_t c, uint32_t b) {
      if (c) {
        x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        const uint32_t k = c & ~LR_SEEN;
        if (k) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)k)), pres);
      }
      if (b) x = __fadd_rn(x, r.bias[b0 + b - 1]);
      if (!(word >> (t & 31) & 1)) x = -INFINITY;
      return Elem<FMT>::store(x);
    };
    auto look = [&](T y, uint32_t t) {
      float v = Elem<FMT>::load(y);
      if (v != v) v = t ? -INFINITY : INFINITY;  // as greta_cuda_argmax
      if (better(v, t, best, bi)) {              // in any order
        best = v;
        bi = t;
      }
    };
    auto single = [&](uint32_t t) {
      uint32_t c = 0, b = 0;
      if (counts) {
        c = table[t - c0];
        if (c) table[t - c0] = 0;
      }
      if (biased) {
        b = biases[t - c0];
        if (b) biases[t - c0] = 0;
      }
      const T y = rule(Elem<FMT>::load(in[t]), t, allowed ? allowed[t / 32] : 0xffffffffu, c, b);
      if (out) out[t] = y;
      look(y, t);
    };
    // Tokens that neither ids nor biases are about need the mask alone.  The others stay as they are for now and are gathered: a division for a lane or two of every
    // warp and token cost more than all the rest (64 rows of 128256: 56 us).
    uint32_t about = 0;      // bits: of the thread's tokens
    float most = -INFINITY;  // of those that are done with; a NaN is none
#pragma unroll
    for (uint32_t k = 0; k < PACKS; ++k) {
      const uint32_t i = k * threads + tid, t = c0 + i * W;
      if (i < whole) {
        uint32_t there[W];
#pragma unroll
        for (uint32_t e = 0; e < W; e += 4) {
          const uint4 x = counts ? *reinterpret_cast<const uint4 *>(table + i * W + e) : make_uint4(0, 0, 0, 0);
          const uint4 y = biased ? *reinterpret_cast<const uint4 *>(biases + i * W + e) : make_uint4(0, 0, 0, 0);
          there[e] = x.x | y.x, there[e + 1] = x.y | y.y, there[e + 2] = x.z | y.z, there[e + 3] = x.w | y.w;
        }
        const uint32_t seen = word[k] >> (t & 31);
#pragma unroll
        for (uint32_t e = 0; e < W; ++e) {
          if (there[e]) {
            about |= 1u << (k * W + e);
          } else {
            if (!(seen >> e & 1)) p[k].x[e] = Elem<FMT>::store(-INFINITY);
            most = fmaxf(most, Elem<FMT>::load(p[k].x[e]));
          }
        }
        if (out) *reinterpret_cast<Pack *>(out + t) = p[k];
      }
    }
    // Where the largest lies is looked for only when it is above all that the warp has seen.  Both zeros are one value: -0 + 0 = +0.
    const uint32_t bits = __float_as_uint(__fadd_rn(most, 0.f)), key = bits ^ ((uint32_t)((int)bits >> 31) | 0x80000000u), highest = __reduce_max_sync(0xffffffffu, key);
    if (highest > above) {
      above = highest;
      if (key == highest) {
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int x = (int)LR_EACH - 1; x >= 0; --x) {
          const uint32_t i = (uint32_t)x / W * threads + tid;
          if (i < whole && !(about >> x & 1) && Elem<FMT>::load(p[x / W].x[x % W]) == most) at = c0 + i * W + (uint32_t)x % W;
        }
        if (at != 0xffffffffu && better(most, at, best, bi)) {
          best = most;
          bi = at;
        }
      }
    }
    if (c0 == 0 && tid == 0 && whole && !(about & 1)) look(p[0].x[0], 0);  // NaN counts in the first place
    if (__any_sync(0xffffffffu, about)) {
      uint32_t before = __popc(about);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= (uint32_t)o) before += x;
      }
      uint32_t at = 0;
      if (lane == 31) at = atomicAdd(&n_later, before);
      at = __shfl_sync(0xffffffffu, at, 31) + before - __popc(about);
      for (; about; about &= about - 1) {
        const uint32_t x = __ffs(about) - 1;
        later[at++] = (uint16_t)((x / W * threads + tid) * W + x % W);
      }
    }
    // what is no whole piece, or rows that do not begin at 16-byte boundaries
    for (uint32_t t = c0 + whole * W + tid; t < c0 + n; t += threads) single(t);
    if (counts || biased) {
      __syncthreads();
      const uint32_t n = n_later;
      for (uint32_t i = tid; i < n; i += threads) single(c0 + later[i]);
      __syncthreads();
      if (tid == 0) n_later = 0;
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
    best = l < threads / 32 ? sv[l] : -INFINITY;
    bi = l < threads / 32 ? si[l] : 0xffffffffu;
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
  // One chunk per CTA where the rows' clusters run at the same time (a GPC holds two of eight CTAs of 1024 threads, four of 512): latency counts.  Else CTAs of 256
  // threads, four an SM, whose phases overlap.  Vocabulary 128256, 4096 ids, 300 biases, masks: 14 rows 10.6 us with 1024 threads, 18 rows 17 with 512 and 23 with 256,
  // 64 rows 35 with 512 and 32 with 256.
  constexpr uint32_t SIZES[2] = {1024, 512};
  static int clusters[64][2] = {};  // 1 + clusters of each size that run at a time
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  for (int i = 0; i < 2; ++i)
    if (!clusters[dev][i]) {
      const uint32_t bytes = (2 * SIZES[i] * LR_EACH + LR_IDS + 2 * LR_BIASES) * 4 + SIZES[i] * LR_EACH * 2;
      if (i == 0) GRETA_CUDA_TRY(cudaFuncSetAttribute(logits_rules_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(8);
      cfg.blockDim = dim3(SIZES[i]);
      cfg.dynamicSmemBytes = bytes;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = 8;
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int n = 0;
      GRETA_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, logits_rules_kernel<FMT>, &cfg));
      clusters[dev][i] = n + 1;
    }
  const uint32_t most = M < (uint32_t)clusters[dev][0] ? SIZES[0] : M < (uint32_t)clusters[dev][1] ? SIZES[1] : 256;
  const uint32_t needed = (((a.V + ctas - 1) / ctas + LR_EACH - 1) / LR_EACH + 31) & ~31u;  // threads that one chunk takes
  const uint32_t threads = std::max(128u, std::min(needed, most)), chunk = threads * LR_EACH;
  const bool counts = a.r.ids && (a.r.repetition || a.r.frequency || a.r.presence);
  const size_t smem = ((size_t)(counts ? chunk + LR_IDS : 0) + (a.r.bias_ids ? chunk + 2 * LR_BIASES : 0)) * 4 + (counts || a.r.bias_ids ? chunk * 2 : 0);
  GRETA_CUDA_TRY(launch_pdl_cluster(logits_rules_kernel<FMT>, dim3(ctas, M), dim3(threads), ctas, smem, stream, a));
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
  GRETA_REQUIRE(!out || out == logits || !rows_meet(logits, (size_t)ld * size, (size_t)V * size, out, (size_t)ld_out * size, (size_t)V * size, M), "%s: out overlaps the logits", name);
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
