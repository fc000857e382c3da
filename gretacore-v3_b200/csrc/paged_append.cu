// New rows of a ragged batch into a paged cache: queries and keys rotated to their positions on the way, keys and values to their pages.
//
// Bytes are what bounds it: q, k and v in, q and the two cache rows out, nothing else.  A CTA takes a token (or a part of its heads where there are few
// tokens): it finds the token's sequence by counting starts, takes the cosines and sines of all pairs once for all heads, then moves
// eight pairs a thread (two 16-byte loads of 16-bit values, four of 32-bit).
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

struct AppendArgs {
  greta_paged_cache c;
  greta_ragged r;
  const void *q, *k, *v;
  void *q_out;
  uint32_t ld_q, ld_k, ld_v, ld_q_out, heads, dims;
  int q_fmt;
  bool interleaved;
  float amplitude;
  uint64_t turn[64];  // 2^64 * freq / (2 pi)
};

template <int FMT>
__device__ __forceinline__ float load1(const void *p, size_t i) {
  if (FMT == GRETA_FMT_F32) return static_cast<const float *>(p)[i];
  if (FMT == GRETA_FMT_F16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
template <int FMT>
__device__ __forceinline__ void load8(const void *p, size_t i, float (&x)[8]) {
  if (FMT == GRETA_FMT_F32) {
    const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i), b = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (FMT == GRETA_FMT_F16) {
        const float2 f = h2_to_f2(w[e]);
        x[2 * e] = f.x, x[2 * e + 1] = f.y;
      } else {
        x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      }
    }
  }
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

// VEC: the rotated part is whole groups of eight pairs (and a head whole groups of eight elements, always).
template <int FMT, bool VEC>
__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ float cs[64], sn[64];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tok = blockIdx.x, tid = threadIdx.x;
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
  const uint32_t d = a.c.dim, half = a.dims / 2, G = a.c.kv_heads;
  if (tid < half) {
    const uint64_t t = (uint64_t)(uint32_t)pos * a.turn[tid];
    float sine, cosine;
    sincospif((float)(int32_t)(t >> 32) * 4.656612873077393e-10f, &sine, &cosine);  // turns in [-1/2, 1/2) times 2, as half turns
    cs[tid] = cosine * a.amplitude;
    sn[tid] = sine * a.amplitude;
  }
  __syncthreads();
  const size_t row = ((size_t)(held ? page : 0) * G * a.c.page + (uint32_t)pos % a.c.page) * d, step = (size_t)a.c.page * d;  // of kv head 0; to the next head
  const uint32_t hq = a.q ? a.heads : 0, at = blockIdx.y * PA_THREADS + tid, all = gridDim.y * PA_THREADS;
  // Heads' units: eight pairs (or one), then eight elements (or one) of the part that is not rotated; all heads of q, then of k.
  const uint32_t turned = VEC ? a.dims / 16 : half, straight = (d - a.dims) / (VEC ? 8 : 1), units = turned + straight;
  for (uint32_t i = at; i < (hq + G) * units; i += all) {
    const uint32_t h = i / units, u = i % units;
    const bool is_q = h < hq;
    const void *src = is_q ? a.q : a.k;
    const size_t from = is_q ? (size_t)tok * a.ld_q + (size_t)h * d : (size_t)tok * a.ld_k + (size_t)(h - hq) * d;
    void *dst = is_q ? a.q_out : a.c.k;
    const size_t to = is_q ? (size_t)tok * a.ld_q_out + (size_t)h * d : row + (h - hq) * step;
    const int fmt = is_q ? a.q_fmt : a.c.fmt;
    if (!is_q && !held) continue;
    if (u < turned) {
      const bool near = a.interleaved;
      if (VEC) {
        const uint32_t e0 = near ? 16 * u : 8 * u, e1 = near ? 16 * u + 8 : half + 8 * u;
        float x[8], y[8];
        load8<FMT>(src, from + e0, x);
        load8<FMT>(src, from + e1, y);
        if (near) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float c0 = cs[8 * u + e], s0 = sn[8 * u + e], c1 = cs[8 * u + 4 + e], s1 = sn[8 * u + 4 + e];
            const float x0 = x[2 * e], x1 = x[2 * e + 1], y0 = y[2 * e], y1 = y[2 * e + 1];
            x[2 * e] = x0 * c0 - x1 * s0, x[2 * e + 1] = x1 * c0 + x0 * s0;
            y[2 * e] = y0 * c1 - y1 * s1, y[2 * e + 1] = y1 * c1 + y0 * s1;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float c = cs[8 * u + e], z = sn[8 * u + e], x0 = x[e], y0 = y[e];
            x[e] = x0 * c - y0 * z, y[e] = y0 * c + x0 * z;
          }
        }
        store8(dst, to + e0, fmt, x);
        store8(dst, to + e1, fmt, y);
      } else {
        const uint32_t e0 = near ? 2 * u : u, e1 = near ? 2 * u + 1 : half + u;
        const float x = load1<FMT>(src, from + e0), y = load1<FMT>(src, from + e1), c = cs[u], z = sn[u];
        store1(dst, to + e0, fmt, x * c - y * z);
        store1(dst, to + e1, fmt, y * c + x * z);
      }
    } else if (VEC) {
      const uint32_t e = a.dims + 8 * (u - turned);
      float x[8];
      load8<FMT>(src, from + e, x);
      store8(dst, to + e, fmt, x);
    } else {
      const uint32_t e = a.dims + (u - turned);
      store1(dst, to + e, fmt, load1<FMT>(src, from + e));
    }
  }
  if (!held) return;
  for (uint32_t i = at; i < G * (d / 8); i += all) {
    const uint32_t h = i / (d / 8), e = i % (d / 8) * 8;
    float x[8];
    load8<FMT>(a.v, (size_t)tok * a.ld_v + (size_t)h * d + e, x);
    store8(a.c.v, row + h * step + e, a.c.fmt, x);
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
  if (rows->tokens == 0) return GRETA_OK;
  // Few tokens: heads spread over more CTAs, down to a unit or two per thread.
  const bool vec = a.dims % 16 == 0;
  const uint32_t units = ((q ? heads : 0) + G) * (vec ? a.dims / 16 + (d - a.dims) / 8 : a.dims / 2 + d - a.dims);
  const uint32_t parts = rows->tokens >= 1024 ? 1 : std::max(1u, std::min({(units + PA_THREADS - 1) / PA_THREADS, 1024 / rows->tokens, 64u}));
  auto go = [&](auto kernel) { return launch_pdl(kernel, dim3(rows->tokens, parts), dim3(PA_THREADS), 0, static_cast<cudaStream_t>(stream), a); };
  if (fmt == GRETA_FMT_F32)
    GRETA_CUDA_TRY(vec ? go(paged_append_kernel<GRETA_FMT_F32, true>) : go(paged_append_kernel<GRETA_FMT_F32, false>));
  else if (fmt == GRETA_FMT_F16)
    GRETA_CUDA_TRY(vec ? go(paged_append_kernel<GRETA_FMT_F16, true>) : go(paged_append_kernel<GRETA_FMT_F16, false>));
  else
    GRETA_CUDA_TRY(vec ? go(paged_append_kernel<GRETA_FMT_BF16, true>) : go(paged_append_kernel<GRETA_FMT_BF16, false>));
  return launched("paged_append_kernel");
}
