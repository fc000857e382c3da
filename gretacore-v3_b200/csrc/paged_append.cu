// New rows of a ragged batch into a paged cache: queries and keys rotated to their positions on the way, keys and values to their pages.
//
// Bytes are what bounds it: q, k and v in, q and the two cache rows out, nothing else.  A CTA takes a token (or a part of its heads where there are few
// tokens): it finds the token's sequence by counting starts, takes the cosines and sines of all pairs once for all heads, then turns
// eight pairs a thread (two 16-byte loads of 16-bit values, four of 32-bit), which were asked for before all that.
//
// The angle of pair i at position p is p * freq_i.  In fp32 it loses a bit for every doubling of p.  Here freq_i / 2 pi is a 64-bit binary fraction of a turn,
// made on the host in extended precision: p times it, modulo 2^64, is the fraction of a turn to p * 2^-65, whole turns fall away for nothing, and its
// upper 32 bits go to sincospi.
#include <math.h>

#include <algorithm>

#include "paged.cuh"

using namespace greta;

namespace {

constexpr uint32_t PA_THREADS = 256;
// Units of a thread that are loaded before anything else, and CTAs a SM that the registers leave room for.  16 bits: three, all of a token of 64 + 8 heads of 128, and
// four CTAs (16384 of them: 128 us, 5.3 TB/s; three CTAs: 148, five: 154; two units and five CTAs: 133).  32 bits: one, and more CTAs (8192 tokens of 32 + 32 heads: 98 us,
// 6.1 TB/s; three: 112).
__host__ __device__ constexpr int pa_ahead(int fmt) { return fmt == GRETA_FMT_F32 ? 1 : 3; }
__host__ __device__ constexpr int pa_ctas(int fmt) { return fmt == GRETA_FMT_F32 ? 6 : 4; }

struct AppendArgs {
  greta_paged_cache c;
  greta_ragged r;
  const void *q, *k, *v;
  void *q_out;
  uint32_t ld_q, ld_k, ld_v, ld_q_out, heads, dims;
  int q_fmt;
  bool interleaved;
  float amplitude;
  uint32_t by_units, by_pieces;  // 2^31 over a head's units and pieces, rounded up: division by multiplication (exact below 2^31 / 16)
  uint64_t turn[64];  // 2^64 * freq / (2 pi)
};

template <int FMT>
__device__ __forceinline__ float load1(const void *p, size_t i) {
  if (FMT == GRETA_FMT_F32) return static_cast<const float *>(p)[i];
  if (FMT == GRETA_FMT_F16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store1(void *p, size_t i, int fmt, float x) {
  if (fmt == GRETA_FMT_F32)
    static_cast<float *>(p)[i] = x;
  else if (fmt == GRETA_FMT_F16)
    static_cast<__half *>(p)[i] = __float2half_rn(x);
  else
    static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}
__device__ __forceinline__ void store8(void *p, size_t i, int fmt, const float (&x)[8]) {
  if (fmt == GRETA_FMT_F32) {
    float4 *d = reinterpret_cast<float4 *>(static_cast<float *>(p) + i);
    d[0] = make_float4(x[0], x[1], x[2], x[3]);
    d[1] = make_float4(x[4], x[5], x[6], x[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (fmt == GRETA_FMT_F16) {
      const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t *>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t *>(&h);
    }
  }
  *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Sixteen values as they lie in memory.
template <int FMT>
struct Raw {
  uint4 w[FMT == GRETA_FMT_F32 ? 4 : 2];
  static constexpr int HALF = FMT == GRETA_FMT_F32 ? 2 : 1;
  __device__ __forceinline__ void load(const void *p, size_t i, int half) {  // eight of them
    const uint4 *src = reinterpret_cast<const uint4 *>(FMT == GRETA_FMT_F32 ? static_cast<const void *>(static_cast<const float *>(p) + i)
                                                                              : static_cast<const void *>(static_cast<const uint16_t *>(p) + i));
#pragma unroll
    for (int j = 0; j < HALF; ++j) w[half * HALF + j] = src[j];
  }
  __device__ __forceinline__ void values(int half, float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < HALF; ++j) {
      const uint4 v = w[half * HALF + j];
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (FMT == GRETA_FMT_F32) {
          x[4 * j + e] = __uint_as_float(u[e]);
        } else if (FMT == GRETA_FMT_F16) {
          const float2 f = h2_to_f2(u[e]);
          x[2 * e] = f.x, x[2 * e + 1] = f.y;
        } else {
          x[2 * e] = __uint_as_float(u[e] << 16), x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
        }
      }
    }
  }
};

// What a thread moves at a time: eight pairs, or (`straight`) eight elements that are not rotated, of a head of q, k or v.
struct Unit {
  uint32_t h, e0, e1;  // head (of q, then of k, then of v); elements
  bool straight;
};

template <int FMT>
__global__ void __launch_bounds__(PA_THREADS, pa_ctas(FMT)) paged_append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int PA_AHEAD = pa_ahead(FMT);
  __shared__ float cs[64], sn[64];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tok = blockIdx.x, tid = threadIdx.x, d = a.c.dim, half = a.dims / 2, G = a.c.kv_heads, hq = a.q ? a.heads : 0;
  const uint32_t first = blockIdx.y * PA_THREADS + tid, step = gridDim.y * PA_THREADS, turned = a.dims / 16, straight = (d - a.dims) / 8, units = turned + straight, pieces = d / 8;
  const uint32_t of_qk = (hq + G) * units, all = of_qk + G * pieces;
  auto unit = [&](uint32_t i) {
    Unit u;
    if (i < of_qk) {
      u.h = __umulhi(2 * i, a.by_units);
      const uint32_t x = i - u.h * units;
      u.straight = x >= turned;
      u.e0 = u.straight ? a.dims + 8 * (x - turned) : a.interleaved ? 16 * x : 8 * x;
      u.e1 = a.interleaved ? 16 * x + 8 : half + 8 * x;
    } else {
      const uint32_t v = __umulhi(2 * (i - of_qk), a.by_pieces);
      u.h = hq + G + v;
      u.straight = true;
      u.e0 = 8 * (i - of_qk - v * pieces);
      u.e1 = 0;
    }
    return u;
  };
  auto load = [&](const Unit &u, Raw<FMT> &r) {
    const void *src = u.h < hq ? a.q : u.h < hq + G ? a.k : a.v;
    const size_t at = u.h < hq ? (size_t)tok * a.ld_q + (size_t)u.h * d : u.h < hq + G ? (size_t)tok * a.ld_k + (size_t)(u.h - hq) * d : (size_t)tok * a.ld_v + (size_t)(u.h - hq - G) * d;
    r.load(src, at + u.e0, 0);
    if (!u.straight) r.load(src, at + u.e1, 1);
  };
  // The first units are on their way while the token's sequence is looked for: neither depends on the other.  (A token behind the last sequence reads its
  // rows of the buffers for nothing.)
  Raw<FMT> raw[PA_AHEAD];
#pragma unroll
  for (int x = 0; x < PA_AHEAD; ++x)
    if (first + x * step < all) load(unit(first + x * step), raw[x]);
  // The token's sequence: the last whose start is at or before it (starts do not decrease; empty ones in between are passed over).
  uint32_t before = 0;
  for (uint32_t b0 = 0;; b0 += PA_THREADS) {
    const uint32_t n = __syncthreads_count(b0 + tid < a.r.batch && __ldcg(a.r.start + b0 + tid) <= tok);
    before += n;
    if (n < PA_THREADS) break;
  }
  if (before == 0) return;
  const uint32_t b = before - 1;
  const PagedSeq s = paged_seq(a.r, a.c.ld_table * a.c.page, b);
  const int pos = s.pos0 + (int)(tok - s.first);
  if (tok - s.first >= s.rows || pos < 0) return;
  const int page = __ldcg(a.c.table + (size_t)b * a.c.ld_table + (uint32_t)pos / a.c.page);
  const bool held = page >= 0 && (uint32_t)page < a.c.pages;
  if (tid < half) {
    const uint64_t t = (uint64_t)(uint32_t)pos * a.turn[tid];
    float sine, cosine;
    sincospif((float)(int32_t)(t >> 32) * 4.656612873077393e-10f, &sine, &cosine);  // turns in [-1/2, 1/2) times 2, as half turns
    cs[tid] = cosine * a.amplitude;
    sn[tid] = sine * a.amplitude;
  }
  __syncthreads();
  const size_t row = ((size_t)(held ? page : 0) * G * a.c.page + (uint32_t)pos % a.c.page) * d, next_head = (size_t)a.c.page * d;  // of KV head 0
  auto store = [&](const Unit &u, const Raw<FMT> &r) {
    const bool is_q = u.h < hq;
    if (!is_q && !held) return;
    void *dst = is_q ? a.q_out : u.h < hq + G ? a.c.k : a.c.v;
    const size_t to = is_q ? (size_t)tok * a.ld_q_out + (size_t)u.h * d : row + (u.h < hq + G ? u.h - hq : u.h - hq - G) * next_head;
    const int fmt = is_q ? a.q_fmt : a.c.fmt;
    float x[8], y[8];
    r.values(0, x);
    if (!u.straight) {
      r.values(1, y);
      const uint32_t p = (a.interleaved ? u.e0 / 16 : u.e0 / 8) * 8;  // its pairs
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float c0 = cs[p + e], s0 = sn[p + e], c1 = cs[p + 4 + e], s1 = sn[p + 4 + e];
          const float x0 = x[2 * e], x1 = x[2 * e + 1], y0 = y[2 * e], y1 = y[2 * e + 1];
          x[2 * e] = x0 * c0 - x1 * s0, x[2 * e + 1] = x1 * c0 + x0 * s0;
          y[2 * e] = y0 * c1 - y1 * s1, y[2 * e + 1] = y1 * c1 + y0 * s1;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float c = cs[p + e], z = sn[p + e], x0 = x[e], y0 = y[e];
          x[e] = x0 * c - y0 * z, y[e] = y0 * c + x0 * z;
        }
      }
      store8(dst, to + u.e1, fmt, y);
    }
    store8(dst, to + u.e0, fmt, x);
  };
#pragma unroll
  for (int x = 0; x < PA_AHEAD; ++x)
    if (first + x * step < all) store(unit(first + x * step), raw[x]);
  for (uint32_t i = first + PA_AHEAD * step; i < all; i += step) {
    const Unit u = unit(i);
    load(u, raw[0]);
    store(u, raw[0]);
  }
}

// The same where the rotated part is no whole groups of eight pairs: a pair or an element at a time.
template <int FMT>
__global__ void __launch_bounds__(PA_THREADS) paged_append_pairs_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ float cs[64], sn[64];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tok = blockIdx.x, tid = threadIdx.x;
  uint32_t before = 0;
  for (uint32_t b0 = 0;; b0 += PA_THREADS) {
    const uint32_t n = __syncthreads_count(b0 + tid < a.r.batch && __ldcg(a.r.start + b0 + tid) <= tok);
    before += n;
    if (n < PA_THREADS) break;
  }
  if (before == 0) return;
  const uint32_t b = before - 1;
  const PagedSeq s = paged_seq(a.r, a.c.ld_table * a.c.page, b);
  const int pos = s.pos0 + (int)(tok - s.first);
  if (tok - s.first >= s.rows || pos < 0) return;
  const int page = __ldcg(a.c.table + (size_t)b * a.c.ld_table + (uint32_t)pos / a.c.page);
  const bool held = page >= 0 && (uint32_t)page < a.c.pages;
  const uint32_t d = a.c.dim, half = a.dims / 2, G = a.c.kv_heads, hq = a.q ? a.heads : 0;
  if (tid < half) {
    const uint64_t t = (uint64_t)(uint32_t)pos * a.turn[tid];
    float sine, cosine;
    sincospif((float)(int32_t)(t >> 32) * 4.656612873077393e-10f, &sine, &cosine);
    cs[tid] = cosine * a.amplitude;
    sn[tid] = sine * a.amplitude;
  }
  __syncthreads();
  const size_t row = ((size_t)(held ? page : 0) * G * a.c.page + (uint32_t)pos % a.c.page) * d, next_head = (size_t)a.c.page * d;
  const uint32_t units = half + d - a.dims;
  for (uint32_t i = blockIdx.y * PA_THREADS + tid; i < (hq + 2 * G) * units; i += gridDim.y * PA_THREADS) {
    const uint32_t h = i / units, u = i % units;
    const bool is_q = h < hq, is_v = h >= hq + G;
    if (!is_q && !held) continue;
    const void *src = is_q ? a.q : is_v ? a.v : a.k;
    const size_t from = is_q ? (size_t)tok * a.ld_q + (size_t)h * d : is_v ? (size_t)tok * a.ld_v + (size_t)(h - hq - G) * d : (size_t)tok * a.ld_k + (size_t)(h - hq) * d;
    void *dst = is_q ? a.q_out : is_v ? a.c.v : a.c.k;
    const size_t to = is_q ? (size_t)tok * a.ld_q_out + (size_t)h * d : row + (is_v ? h - hq - G : h - hq) * next_head;
    const int fmt = is_q ? a.q_fmt : a.c.fmt;
    if (u < half) {
      const uint32_t e0 = a.interleaved ? 2 * u : u, e1 = a.interleaved ? 2 * u + 1 : half + u;
      const float x = load1<FMT>(src, from + e0), y = load1<FMT>(src, from + e1), c = is_v ? 1.f : cs[u], z = is_v ? 0.f : sn[u];
      store1(dst, to + e0, fmt, is_v ? x : x * c - y * z);
      store1(dst, to + e1, fmt, is_v ? y : y * c + x * z);
    } else {
      const uint32_t e = a.dims + (u - half);
      store1(dst, to + e, fmt, load1<FMT>(src, from + e));
    }
  }
}

}  // namespace

extern "C" int greta_cuda_paged_append(greta_stream_t stream, const greta_paged_cache *cache, const greta_ragged *rows, const greta_rotation *rotation, int fmt,
                                       const void *q, uint32_t ld_q, const void *k, uint32_t ld_k, const void *v, uint32_t ld_v, uint32_t heads, void *q_out,
                                       int q_fmt, uint32_t ld_q_out) {
  if (int rc = paged_check(cache, rows, "paged_append")) return rc;
  const uint32_t d = cache->dim, G = cache->kv_heads;
  GRETA_REQUIRE(rotation && k && v && !q == !q_out, "paged_append: null pointer");
  GRETA_REQUIRE(paged_float(fmt) && (!q || paged_float(q_fmt)), "paged_append: formats %d and %d, not fp32, fp16 or bf16", fmt, q_fmt);
  GRETA_REQUIRE(rotation->dims <= d && rotation->dims % 2 == 0, "paged_append: rotation of %u of %u elements", rotation->dims, d);
  GRETA_REQUIRE(!q || (heads >= 1 && heads <= 65535), "paged_append: %u heads", heads);
  GRETA_REQUIRE(ld_k >= G * d && ld_v >= G * d && (!q || (ld_q >= heads * d && ld_q_out >= heads * d)), "paged_append: rows closer than their elements");
  auto whole = [](const void *p, uint32_t ld, int f) { return aligned16(p) && (size_t)ld * paged_size(f) % 16 == 0; };
  GRETA_REQUIRE(whole(k, ld_k, fmt) && whole(v, ld_v, fmt) && (!q || (whole(q, ld_q, fmt) && whole(q_out, ld_q_out, q_fmt))),
                "paged_append: rows that do not begin at 16-byte boundaries");
  GRETA_REQUIRE(q != q_out || !q || (fmt == q_fmt && ld_q == ld_q_out), "paged_append: in place between two types or row lengths");
  AppendArgs a{};
  a.c = *cache;
  a.r = *rows;
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.ld_q = ld_q, a.ld_k = ld_k, a.ld_v = ld_v, a.ld_q_out = ld_q_out;
  a.heads = heads;
  a.dims = rotation->dims;
  a.q_fmt = q_fmt;
  a.interleaved = rotation->interleaved != 0;
  a.amplitude = rotation->amplitude;
  GRETA_REQUIRE(a.dims == 0 || rotation->freq || (rotation->base > 0 && std::isfinite(rotation->base)), "paged_append: base %g", rotation->base);
  // Powers of base^(-2 / dims) by products: 63 roundings to 64 bits, and one powl instead of 64 (18 us of a call).
  const long double step = a.dims && !rotation->freq ? powl((long double)rotation->base, -2.0L / a.dims) : 1.0L;
  long double power = 1.0L;
  for (uint32_t i = 0; i < a.dims / 2; ++i) {
    const long double f = rotation->freq ? (long double)rotation->freq[i] : power;
    power *= step;
    GRETA_REQUIRE(std::isfinite((double)f), "paged_append: frequency %u is no finite number", i);
    const long double turns = f / 6.283185307179586476925286766559005768L, part = turns - floorl(turns);  // of a turn per position, 0 .. 1
    const long double scaled = part * 18446744073709551616.0L + 0.5L;
    a.turn[i] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
  }
  auto over = [&](const void *p, uint32_t ld, uint32_t n) {
    return rows_meet(p, (size_t)ld * paged_size(fmt), (size_t)n * d * paged_size(fmt), q_out, (size_t)ld_q_out * paged_size(q_fmt), (size_t)heads * d * paged_size(q_fmt), rows->tokens);
  };
  GRETA_REQUIRE(!q || !((q != q_out && over(q, ld_q, heads)) || over(k, ld_k, G) || over(v, ld_v, G)), "paged_append: q_out overlaps q, k or v");
  if (rows->tokens == 0) return GRETA_OK;
  // Few tokens: heads spread over more CTAs, down to a unit or two per thread.
  const bool vec = a.dims % 16 == 0;
  const uint32_t units = vec ? ((q ? heads : 0) + G) * (a.dims / 16 + (d - a.dims) / 8) + G * d / 8 : ((q ? heads : 0) + 2 * G) * (d - a.dims / 2);
  if (vec) {
    auto by = [](uint32_t n) { return (0x80000000u + n - 1) / n; };
    a.by_units = by(a.dims / 16 + (d - a.dims) / 8);
    a.by_pieces = by(d / 8);
  }
  const uint32_t parts = rows->tokens >= 1024 ? 1 : std::max(1u, std::min({(units + PA_THREADS - 1) / PA_THREADS, 1024 / rows->tokens, 64u}));
  auto go = [&](auto kernel) { return launch_pdl(kernel, dim3(rows->tokens, parts), dim3(PA_THREADS), 0, static_cast<cudaStream_t>(stream), a); };
  if (fmt == GRETA_FMT_F32)
    GRETA_CUDA_TRY(vec ? go(paged_append_kernel<GRETA_FMT_F32>) : go(paged_append_pairs_kernel<GRETA_FMT_F32>));
  else if (fmt == GRETA_FMT_F16)
    GRETA_CUDA_TRY(vec ? go(paged_append_kernel<GRETA_FMT_F16>) : go(paged_append_pairs_kernel<GRETA_FMT_F16>));
  else
    GRETA_CUDA_TRY(vec ? go(paged_append_kernel<GRETA_FMT_BF16>) : go(paged_append_pairs_kernel<GRETA_FMT_BF16>));
  return launched("paged_append_kernel");
}
