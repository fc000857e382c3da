// Attention of a ragged batch's new rows over a paged cache on the 5th-generation tensor cores: portions of prompts, queries of the cache's type.
//
// A CTA takes a block of 256 query rows of one KV head as two tiles of 128: row R of a sequence and KV head is token R / group, head R % group, so a tile
// is 128 / group tokens with all their heads and every key tile is fetched once for them.  Keys come in tiles of 128, page by page, by TMA (a page's rows of a head
// are contiguous); queries by TMA as boxes of [tokens][group][64].
//   warp 0: copies, and zeros over what the last page holds behind the sequence's end; warp 1: MMAs; warps 2-9 and 10-17: the rows of the first and
//   second tile, two threads each (64 keys of a tile, half of the outputs): maxima, probabilities, outputs.
// The two tiles take turns: while the tensor core multiplies one (P V of this key tile, Q K of the next), the other's probabilities are made.
//   tensor memory: scores of tile A and B at columns 0 and 128, each half of which is overwritten by its probabilities (32 columns), outputs at 256 and 384.
// A row's sums are rescaled only when its maximum has grown by more than 2^8 (probabilities up to 2^8 fit every type); the scores' barrier of a key tile says that
// the products of the one before are in, so the rows' own threads do that.
#include <math.h>

#include <algorithm>

#include "mma_device.cuh"
#include "paged_attention.cuh"
#include "tc_device.cuh"

using namespace greta;

namespace {

constexpr uint32_t PT_ROWS = 128, PT_KEYS = 128, PT_THREADS = 576, PT_UNITS = 5, PT_TMEM = 512;
constexpr uint32_t PT_SLAB = 128 * 128;  // bytes of 64 elements of 128 rows
constexpr int PT_EMULATED = 1;           // pairs of probabilities out of four that the FMA units make: the special-function unit's 16 a clock bound the tile otherwise
constexpr float PT_LAZY = 8.f;           // log2 of what a row's maximum may grow by before its sums are rescaled
constexpr float PT_LOWEST = -3.4028234e38f;  // a row's maximum before any score

__device__ __forceinline__ void tma_load_3d(void *smem_dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(smem_dst)),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
               : "memory");
}
// On the critical path: waits that the hardware ends (a time hint wakes late; testing without rest takes issue slots from the warps that compute).
__device__ __noinline__ bool poll_slow(uint32_t bar, uint32_t parity, volatile int *abort_flag, int code) {
  const long long t0 = clock64();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    if (clock64() - t0 > WAIT_LIMIT_CYCLES) {
      *abort_flag = code;
      return false;
    }
  }
}
__device__ __forceinline__ bool poll(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  return poll_slow(smem_u32(bar), parity, abort_flag, code);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (!BF16) return half2_bits(a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of two values without the special-function unit: x = n + r, n an integer (by adding 1.5 * 2^23, whose last place is one) and |r| <= 1/2; a polynomial in r of
// degree 3, fitted to the smallest largest relative error over that interval (7.5e-5, a quarter of half a step of fp16); n is added to its exponent.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  const uint64_t big = pair(12582912.f, 12582912.f);
  const float2 f = unpair(x);
  x = pair(fmaxf(f.x, -126.f), fmaxf(f.y, -126.f));
  const uint64_t t = add2(x, big), n = add2(t, pair(-12582912.f, -12582912.f)), r = fma2(n, pair(-1.f, -1.f), x);
  uint64_t p = fma2(r, pair(0.0551716685f, 0.0551716685f), pair(0.242611125f, 0.242611125f));
  p = fma2(p, r, pair(0.693260968f, 0.693260968f));
  p = fma2(p, r, pair(0.999928057f, 0.999928057f));
  const float2 y = unpair(p), e = unpair(t);
  return pair(__int_as_float(__float_as_int(y.x) + (__float_as_int(e.x) << 23)), __int_as_float(__float_as_int(y.y) + (__float_as_int(e.y) << 23)));
}

// A block of rows of one sequence and KV head, and the key tiles of its two halves.
struct Block {
  uint32_t b, g, token0, t0, t1;      // tiles t0 .. t1 - 1 of either half
  uint32_t tokens[2], lo[2], hi[2];   // of half i: its tokens, tiles lo .. hi - 1
  PagedSeq s;
};

template <int SD, bool BF16>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_tc_kernel(const __grid_constant__ PagedAttnArgs w) {
  constexpr uint32_t DH = SD * 64, UNIT = SD * PT_SLAB;
  extern __shared__ __align__(1024) uint8_t paged_tc_smem[];  // alignment of the swizzled tiles; there is no room to align it by hand
  uint8_t *smem = paged_tc_smem;
  uint8_t *qs = smem, *ring = qs + 2 * UNIT;  // queries of both tiles; keys and values in turn
  uint64_t *bars = reinterpret_cast<uint64_t *>(ring + PT_UNITS * UNIT);
  uint64_t *full = bars, *empty = full + PT_UNITS, *qf = empty + PT_UNITS, *sf = qf + 1, *pf = sf + 2, *vl = pf + 4, *vz = vl + 1, *fin = vz + 1;  // vl: the last values have come; vz: and hold zeros behind the sequence
  float *meet = reinterpret_cast<float *>(fin + 2);  // [tile][half][row]: what the two threads of a row tell each other
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(meet + 4 * PT_ROWS), *place = tmem_slot + 1;  // place: sequence, block
  volatile int *abort_flag = reinterpret_cast<volatile int *>(place + 2);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t group = w.group, TT = PT_ROWS / group;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < PT_UNITS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(qf, 1);
    mbar_init(vl, 1);
    mbar_init(vz, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sf[i], 1);
      mbar_init(&pf[2 * i], 8);  // the first and the second 32 keys of both warps of a row
      mbar_init(&pf[2 * i + 1], 8);
      mbar_init(&fin[i], 1);
    }
    place[0] = 0xffffffffu;
    *abort_flag = smem_u32(smem) % 1024 ? 999 : 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w.k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w.v) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w.qm) : "memory");
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, PT_TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();

  // ---- which block: sequences in order, the last rows of each (the longest) first, KV heads side by side
  const uint32_t max_len = w.c.ld_table * w.c.page, heads_kv = w.c.kv_heads;
  if (warp == 0 && *abort_flag == 0) {
    uint32_t before = 0;
    const uint32_t mine = blockIdx.x / heads_kv;
    for (uint32_t b0 = 0; b0 < w.r.batch; b0 += 32) {
      uint32_t n = 0;
      if (b0 + lane < w.r.batch) n = (paged_seq(w.r, max_len, b0 + lane).rows + 2 * TT - 1) / (2 * TT);
      uint32_t v = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      if (mine >= before + v - n && mine < before + v) {
        place[0] = b0 + lane;
        place[1] = before + v - 1 - mine;
      }
      before += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  Block k;
  k.b = place[0];
  if (k.b != 0xffffffffu) {
    k.g = blockIdx.x % heads_kv;
    k.s = paged_seq(w.r, max_len, k.b);
    k.token0 = place[1] * 2 * TT;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t first = k.token0 + i * TT;
      k.tokens[i] = first < k.s.rows ? min(TT, k.s.rows - first) : 0;
      const int pos = k.s.pos0 + (int)first, end = pos + (int)k.tokens[i];  // positions pos .. end - 1
      const int from = w.window ? pos - (int)w.window + 1 : 0;
      k.lo[i] = k.tokens[i] == 0 ? k.lo[0] : from > 0 ? (uint32_t)from / PT_KEYS : 0;
      k.hi[i] = k.tokens[i] && end > 0 ? ((uint32_t)end + PT_KEYS - 1) / PT_KEYS : k.lo[i];
    }
    // The second half's tiles begin and end no earlier than the first's, and there is none between them: its first row follows the first half's last.
    k.t0 = k.lo[0];
    k.t1 = max(k.hi[0], k.hi[1]);
    const int last = k.s.pos0 + (int)k.s.rows;  // behind the sequence's last position
    const bool ragged = k.t1 > k.t0 && (int)(k.t1 * PT_KEYS) > last;  // its last tile holds rows behind it

    const bool leader = elect_one();
    if (warp == 0) {
      const uint32_t box = min(w.c.page, PT_KEYS), boxes = PT_KEYS / box;
      const int32_t *table = w.c.table + (size_t)k.b * w.c.ld_table;
      uint32_t it = 0;
      bool ok = true;
      if (leader) {
        mbar_arrive_expect_tx(qf, (k.tokens[1] ? 2 : 1) * SD * 128 * group * TT);
        for (uint32_t i = 0; i < 2; ++i)
          for (uint32_t c = 0; c < SD && k.tokens[i]; ++c)
            tma_load_3d(qs + i * UNIT + c * PT_SLAB, &w.qm, (int)(c * 64), (int)(k.g * group), (int)(k.s.first + k.token0 + i * TT), qf);
      }
      auto page_of = [&](uint32_t t) {
        const uint32_t p = t * PT_KEYS + lane * box;
        return lane < boxes && t < k.t1 && p < k.s.len ? __ldcg(table + p / w.c.page) : -1;
      };
      int next = page_of(k.t0);
      for (uint32_t t = k.t0; t < k.t1; ++t) {
        const int id = next;
        next = page_of(t + 1);
        const uint32_t p = t * PT_KEYS + lane * box;
        // no page: rows in front of the pool, which read as zeros
        const int row = (uint32_t)id < w.c.pages ? (int)(((uint32_t)id * heads_kv + k.g) * w.c.page + p % w.c.page) : -(int)PT_KEYS;
#pragma unroll
        for (uint32_t kv = 0; kv < 2; ++kv, ++it) {
          const uint32_t st = it % PT_UNITS;
          if (ok) ok = poll(&empty[st], ((it / PT_UNITS) & 1) ^ 1, abort_flag, 900 + st);
          __syncwarp();
          uint64_t *bar = kv && ragged && t + 1 == k.t1 ? vl : &full[st];
          if (leader && ok) mbar_arrive_expect_tx(bar, UNIT);
          __syncwarp();
          if (ok && lane < boxes)
            for (uint32_t c = 0; c < SD; ++c) tma_load_2d(ring + st * UNIT + c * PT_SLAB + lane * box * 128, kv ? &w.v : &w.k, (int)(c * 64), row, bar);
        }
      }
      if (ragged) {  // what the last page holds behind the sequence's end: zeros
        if (ok) ok = mbar_wait(vl, 0, abort_flag, 950);
        __syncwarp();
        const uint32_t from = (uint32_t)max(0, last - (int)((k.t1 - 1) * PT_KEYS));
        if (ok) {
          for (uint32_t i = lane; i < (PT_KEYS - from) * 8 * SD; i += 32)
            *reinterpret_cast<uint4 *>(ring + (it - 1) % PT_UNITS * UNIT + i / ((PT_KEYS - from) * 8) * PT_SLAB + from * 128 + i % ((PT_KEYS - from) * 8) * 16) =
                make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
        if (leader && ok) mbar_arrive(vz);
      }
      if (leader && *abort_flag) drain_copies(full, it, PT_UNITS);
      if (leader && *abort_flag) drain_copies(qf, 1, 1);
      if (leader && *abort_flag) drain_copies(vl, ragged ? 1 : 0, 1);
    } else if (warp == 1) {
      constexpr uint32_t idesc_s = BF16 ? instr_desc_bf16(PT_ROWS, PT_KEYS) : instr_desc_f16(PT_ROWS, PT_KEYS);
      constexpr uint32_t idesc_o = (BF16 ? instr_desc_bf16(PT_ROWS, DH) : instr_desc_f16(PT_ROWS, DH)) | (1u << 16);  // values: keys are the rows of memory (N-major operand)
      const uint32_t q_lo = smem_desc_lo(smem_u32(qs)), k_lo = smem_desc_lo(smem_u32(ring));
      const uint32_t v_lo = ((smem_u32(ring) >> 4) & 0x3FFFu) | ((PT_SLAB >> 4) << 16);  // 64-element groups are a slab apart
      bool ok = true;
      if (ok) ok = mbar_wait(qf, 0, abort_flag, 910);
      __syncwarp();
      auto scores = [&](uint32_t i, uint32_t t) {  // of half i with key tile t
        if (leader && ok) {
          tc_fence_after();
          const uint32_t st = 2 * (t - k.t0) % PT_UNITS;
#pragma unroll
          for (uint32_t k16 = 0; k16 < DH / 16; ++k16)
            umma_f16(tmem + i * 128, q_lo + (i * UNIT + (k16 / 4) * PT_SLAB) / 16 + (k16 & 3) * 2, k_lo + (st * UNIT + (k16 / 4) * PT_SLAB) / 16 + (k16 & 3) * 2,
                     SMEM_DESC_HI_SW128, idesc_s, k16 ? 1u : 0u);
          umma_commit(&sf[i]);
        }
      };
      uint32_t np[2] = {0, 0};  // key tiles whose products with the values are under way
      for (uint32_t t = k.t0; t <= k.t1; ++t) {
        // outputs of tile t - 1, scores of tile t, half by half
        const uint32_t ik = 2 * (t - k.t0), iv = 2 * (t - 1 - k.t0) + 1;
        const bool kt = t < k.t1, vt = t > k.t0;
        bool have_k = false, have_v = false;
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          if (vt && t - 1 >= k.lo[i] && t - 1 < k.hi[i]) {
            if (!have_v) {
              if (ok) ok = ragged && t == k.t1 ? poll(vz, 0, abort_flag, 921) : poll(&full[iv % PT_UNITS], (iv / PT_UNITS) & 1, abort_flag, 920);
              have_v = true;
            }
#pragma unroll
            for (uint32_t part = 0; part < 2; ++part) {
              if (ok) ok = poll(&pf[2 * i + part], np[i] & 1, abort_flag, 930 + 2 * i + part);
              __syncwarp();
              if (leader && ok) {
                tc_fence_after();
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) {
                  const uint32_t k16 = (x >> 1) * 4 + part * 2 + (x & 1);  // a half's probabilities lie in the first 32 of its own 64 columns of scores
                  umma_f16_ts(tmem + 256 + i * 128, tmem + i * 128 + (x >> 1) * 64 + (part * 2 + (x & 1)) * 8, v_lo + (iv % PT_UNITS) * (UNIT / 16) + k16 * (2048 >> 4),
                              SMEM_DESC_HI_SW128, idesc_o, (np[i] | part | x) ? 1u : 0u);
                }
              }
            }
            if (leader && ok) {
              if (t == k.hi[i]) umma_commit(&fin[i]);
            }
            ++np[i];
          }
          if (kt && t >= k.lo[i] && t < k.hi[i]) {
            if (!have_k) {
              if (ok) ok = poll(&full[ik % PT_UNITS], (ik / PT_UNITS) & 1, abort_flag, 940);
              have_k = true;
            }
            __syncwarp();
            scores(i, t);
          }
        }
        // every tile has a half that uses it, so both units have been waited for
        if (leader && ok && vt) umma_commit(&empty[iv % PT_UNITS]);
        if (leader && ok && kt) umma_commit(&empty[ik % PT_UNITS]);
      }
    } else {
      const uint32_t i = (uint32_t)(warp - 2) >> 3, half = ((uint32_t)(warp - 2) >> 2) & 1, quad = warp & 3, row = quad * 32 + lane;
      const uint32_t lanes = tmem + (quad * 32 << 16), sb = lanes + i * 128 + half * 64, ob = lanes + 256 + i * 128 + half * (DH / 2);
      float *mine = meet + (i * 2 + half) * PT_ROWS + row, *theirs = meet + (i * 2 + (half ^ 1)) * PT_ROWS + row;
      auto meet_other = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + i * 4 + quad) : "memory"); };  // with the other warp of these rows
      auto agree = [&](bool x) {  // whether any thread of the two warps says so
        uint32_t any;
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"(1 + i * 4 + quad), "r"((uint32_t)x) : "memory");
        return any != 0;
      };
      const bool live = row < k.tokens[i] * group, any_live = quad * 32 < k.tokens[i] * group;
      const uint32_t token = k.token0 + i * TT + row / group;
      const int pos = k.s.pos0 + (int)token;
      const int lim1 = live ? pos + 1 : 0, lim0 = w.window && pos >= (int)w.window ? pos - (int)w.window + 1 : 0;
      // tiles that every live row sees whole need no masks
      const int pos_lo = k.s.pos0 + (int)(k.token0 + i * TT), pos_hi = pos_lo + (int)k.tokens[i] - 1;
      const int whole0 = w.window ? max(0, pos_hi - (int)w.window + 1) : 0, whole1 = pos_lo + 1;
      float m2 = PT_LOWEST, l = 0.f;  // the row's maximum times scale2; the sum of this thread's half
      bool ok = true;
      uint32_t n = 0;
      for (uint32_t t = k.lo[i]; t < k.hi[i]; ++t, ++n) {  // to the end, whatever became of a wait: the two warps of a row meet in every tile
        if (ok) ok = __all_sync(0xffffffffu, poll(&sf[i], n & 1, abort_flag, 960 + i));
        tc_fence_after();
        if (!any_live) {  // rows behind the last: their probabilities may be anything
          if (lane == 0) {
            mbar_arrive(&pf[2 * i]);
            mbar_arrive(&pf[2 * i + 1]);
          }
          continue;
        }
        const int k0 = (int)(t * PT_KEYS);
        const bool masks = k0 < whole0 || k0 + (int)PT_KEYS > whole1;
        uint32_t v[2][32];
        auto hide = [&](int c) {  // scores of keys that the row does not see
          if (masks) {
            const int a = k0 + (int)half * 64 + c * 32, n0 = min(max(lim0 - a, 0), 32), n1 = min(max(lim1 - a, 0), 32);
            const uint32_t seen = (uint32_t)((1ull << n1) - 1) & ~(uint32_t)((1ull << n0) - 1);
            if (!__all_sync(0xffffffffu, seen == 0xffffffffu)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!(seen >> j & 1)) v[c][j] = 0xFF800000u;
            }
          }
        };
        auto largest = [&](int c) {
          float tm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 32; j += 2) tm[(j / 2) & 3] = fmaxf(fmaxf(tm[(j / 2) & 3], __uint_as_float(v[c][j])), __uint_as_float(v[c][j + 1]));
          return fmaxf(fmaxf(tm[0], tm[1]), fmaxf(tm[2], tm[3]));
        };
        uint32_t p[16];
        float sum;
        auto probabilities = [&](int c) {  // p and their sum
          uint64_t two[2] = {0, 0};
          const uint64_t scale = pair(w.scale2, w.scale2), minus = pair(-m2, -m2);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            uint64_t x = fma2(pair(__uint_as_float(v[c][2 * j]), __uint_as_float(v[c][2 * j + 1])), scale, minus);
            if ((j & 3) < PT_EMULATED) {
              x = exp2_pair(x);
            } else {
              const float2 f = unpair(x);
              x = pair(ex2(f.x), ex2(f.y));
            }
            two[j & 1] = add2(two[j & 1], x);
            const float2 f = unpair(x);
            p[j] = pack2<BF16>(f.x, f.y);
          }
          const float2 s0 = unpair(two[0]), s1 = unpair(two[1]);
          sum = (s0.x + s0.y) + (s1.x + s1.y);
        };
        auto release = [&](int c) {  // the products of the first 32 keys begin while the others' probabilities are made
          tmem_st16(sb + c * 16, p);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pf[2 * i + c]);
        };
        // The first 32 probabilities are made against the maximum so far, beside the search for the tile's; where it has grown too much (a row's two
        // threads have to agree, and the barrier tells both) they are made again.
        tmem_ld32(sb, v[0]);
        tmem_ld_wait();
        tmem_ld32(sb + 32, v[1]);
        hide(0);
        float tmax = largest(0);
        probabilities(0);
        tmem_ld_wait();
        hide(1);
        tmax = fmaxf(tmax, largest(1));
        if (agree(n == 0 || tmax * w.scale2 > m2 + PT_LAZY)) {
          *mine = tmax;
          meet_other();
          const float nm = fmaxf(m2, fmaxf(tmax, *theirs) * w.scale2);
          const bool grown = n == 0 || nm > m2 + PT_LAZY;
          const float f = grown ? ex2(m2 - nm) : 1.f;
          if (grown) m2 = nm;
          l *= f;
          if (n) {
#pragma unroll 1
            for (uint32_t c = 0; c < DH / 2; c += 16) {
              tmem_ld16(ob + c, p);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) p[j] = __float_as_uint(__uint_as_float(p[j]) * f);
              tmem_st16(ob + c, p);
            }
          }
          tmem_ld32(sb, v[0]);
          tmem_ld_wait();
          hide(0);
          probabilities(0);
        }
        l += sum;
        release(0);
        probabilities(1);
        l += sum;
        release(1);
      }
      if (ok && n) ok = __all_sync(0xffffffffu, poll(&fin[i], 0, abort_flag, 970 + i));
      if (any_live) {
        meet_other();  // the last maximum has been read
        *mine = l;
        meet_other();
        l += *theirs;
      }
      if (any_live) {
        // Outputs go through shared memory (the tile's queries have been used): 16 bytes a lane straight from a row per lane are a line each, and took 5 us
        // of a block, 6 more until they had drained and the next block could begin.
        tc_fence_after();
        uint8_t *stage = qs + i * UNIT;
        const float inv = m2 == PT_LOWEST ? 0.f : 1.f / l;  // a row that has seen no score: zeros (its sum holds what 2^-126 is for minus infinity)
        if (ok && n) {
#pragma unroll 1
          for (uint32_t c = half * (DH / 2); c < (half + 1) * (DH / 2); c += 32) {
            uint32_t o[32];
            __syncwarp();
            tmem_ld32(lanes + 256 + i * 128 + c, o);
            tmem_ld_wait();
            float y[32], z = 0.f;  // z: 0, or NaN
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              y[j] = __uint_as_float(o[j]);
              z = fmaf(y[j], 0.f, z);
            }
            if (z != 0.f && live && isfinite(l)) {
              float x[32];  // in memory, which `y` stays out of
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = y[j];
              paged_again<32>(w, BF16, false, k.b, k.s, k.g, (k.token0 + i * TT) * group + row, [&](int j) { return c + j; }, max(lim0, (int)(k.lo[i] * PT_KEYS)), lim1, m2, x);
#pragma unroll
              for (int j = 0; j < 32; ++j) y[j] = x[j];
            }
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              *reinterpret_cast<uint4 *>(stage + row * (DH * 2) + (((c + j) / 8 ^ (row & 7)) << 4)) =
                  make_uint4(pack2<BF16>(y[j] * inv, y[j + 1] * inv), pack2<BF16>(y[j + 2] * inv, y[j + 3] * inv), pack2<BF16>(y[j + 4] * inv, y[j + 5] * inv),
                             pack2<BF16>(y[j + 6] * inv, y[j + 7] * inv));
          }
        }
        meet_other();
        constexpr uint32_t LPR = DH / 8, RPP = 32 / LPR;  // lanes per row, rows per pass
        const uint32_t e = lane % LPR, rows = k.tokens[i] * group;
        if (ok && e * 8 < w.c.dim) {
#pragma unroll 4
          for (uint32_t x = 0; x < 16; x += RPP) {
            const uint32_t r = quad * 32 + half * 16 + x + lane / LPR;
            if (r >= rows) continue;
            uint16_t *out = static_cast<uint16_t *>(w.o) + (size_t)(k.s.first + k.token0 + i * TT + r / group) * w.ld_o + (size_t)(k.g * group + r % group) * w.c.dim;
            *reinterpret_cast<uint4 *>(out + e * 8) = n ? *reinterpret_cast<const uint4 *>(stage + r * (DH * 2) + ((e ^ (r & 7)) << 4)) : make_uint4(0, 0, 0, 0);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) atomicCAS(w.error, 0, *abort_flag);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, PT_TMEM);
  }
}

template <int SD, bool BF16>
int launch_tc(cudaStream_t stream, const PagedAttnArgs &w, uint32_t blocks) {
  constexpr size_t smem = (size_t)(2 + PT_UNITS) * SD * PT_SLAB + (2 * PT_UNITS + 11) * 8 + 4 * PT_ROWS * 4 + 16;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    GRETA_CUDA_TRY(cudaFuncSetAttribute(paged_tc_kernel<SD, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  GRETA_CUDA_TRY(launch_pdl(paged_tc_kernel<SD, BF16>, dim3(blocks * w.c.kv_heads), dim3(PT_THREADS), smem, stream, w));
  return launched("paged_tc_kernel");
}

}  // namespace

namespace greta {

// Queries of the cache's type, groups of up to 128; w.k and w.v with boxes of min(page, 128) rows.
int paged_attn_tc(cudaStream_t stream, PagedAttnArgs &w, uint32_t heads) {
  EncodeTiledFn enc = encode_tiled();
  const uint32_t d = w.c.dim, TT = PT_ROWS / w.group;
  const cuuint64_t dims[3] = {d, heads, w.r.tokens}, strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)w.ld_q * 2};
  const cuuint32_t box[3] = {64, w.group, TT}, one[3] = {1, 1, 1};
  const bool bf16 = w.c.fmt == GRETA_FMT_BF16;
  const CUresult r = enc(&w.qm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(w.q), dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("paged_attn: cuTensorMapEncodeTiled failed with code %d", (int)r);
    return GRETA_ERR_INVALID_ARGS;
  }
  const uint32_t blocks = w.r.tokens / (2 * TT) + std::min(w.r.batch, w.r.tokens);  // no sequence has more than its whole blocks and one
  GRETA_REQUIRE((uint64_t)blocks * w.c.kv_heads < (1ull << 31), "paged_attn: %u blocks of %u heads", blocks, w.c.kv_heads);
  if (d > 64) return bf16 ? launch_tc<2, true>(stream, w, blocks) : launch_tc<2, false>(stream, w, blocks);
  return bf16 ? launch_tc<1, true>(stream, w, blocks) : launch_tc<1, false>(stream, w, blocks);
}

}  // namespace greta
