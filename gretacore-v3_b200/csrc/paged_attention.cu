// Attention of a ragged batch's new rows over a paged cache, few query rows per sequence: the form for single tokens and drafts, and for fp32 queries.
//
// Bytes are what bounds it: every key and value once.  The work is a list of key tiles of 64 (one KV head of one sequence, 16 MT query rows of its
// group: row R of a sequence and group is token R / group, head R % group), cut into one equal share per CTA whatever the sequences' lengths are; a
// row block whose tiles fall to several CTAs is joined by the last of them to finish, in the order of the tiles.  A warp of its own
// fetches pages by TMA (rows of a head in a page are contiguous: one box of up to 64 rows per 64 elements) into a ring; four warps compute:
//   scores: each warp 16 keys, all rows (mma.sync, keys by ldmatrix); the tile's row maxima meet in shared memory;
//   probabilities go to shared memory; values: each warp a quarter of the head's elements, all 64 keys.
// So the outputs are spread over the warps by columns, and nothing is merged when a row block ends.
//
// fp32 queries and probabilities travel as two fp16 or three bf16 values each (of the cache's type, which is exact), products are exact in the fp32
// accumulators: 22 or 24 bits are kept.  16-bit queries are used as they are, probabilities are rounded to 16 bits (half a step: 2^-11 or 2^-8 of each, the sum of
// them is taken in fp32 of the unrounded values).
// fp16 has no steps below 2^-24: probabilities are made 2^15 times as large for it (sums too, so the division at the end takes it out).  Weights down to 2^-18 of a row's
// largest keep 22 bits then, single ones down to 2^-29 their 11, and what is smaller is off by at most 2^-40 of the largest.  (4096 keys behind one of no value and a score 12 or 14
// higher, error of fp32 calls of the outputs' size: 5.8e-7 and 7.0e-7; with probabilities of their own size 3.2e-4 and 1.9e-3.)
//
// 16 sequences around 4096 positions, 64 heads over 8 of 128, fp32 queries: 58 us (4.7 TB/s); 32 of them: 99 us (5.4 TB/s); one sequence of 577, 32 heads: 13.0 us.
// In front of the stream lie 2 us until the shares are known and 4.5 until the first tiles are in (table entry, then page, from all SMs at once), behind it 4 of
// tickets and joining, and SMs are served unevenly: equal shares end 50 to 66 us after the start.  Two CTAs of three stages an SM keep 192 KB on their way; three of two do no better.
// Where two do not fit, one keeps 96 KB: heads above 64, fp32 queries over bf16 from 16 sequences on (the third term's memory; 16 around 4096: 108 us), over fp16 from 112 (96 of 1000: 85 us,
// 128: 165), 16 bits from 379 (128 of 1000: 95 us, 512: 506).
// 64 rows a block in place of 16 for more queries: their operands come from shared memory again for every tile (fp32, prompt of 2048, 32 heads: 969 us over fp16, 1198 over bf16).
#include <math.h>

#include <algorithm>

#include "mma_device.cuh"
#include "paged_attention.cuh"

#include "tc_device.cuh"

using namespace greta;

namespace {

constexpr uint32_t PM_KEYS = 64, PM_WARPS = 4, PM_THREADS = 32 * (PM_WARPS + 1);
constexpr uint32_t PM_LIST = 4;  // what a row block costs besides its tiles, in tiles: its queries, sums and outputs (one sequence in ten of one tile, 96 in all: 65.4 us; 2: 66.2)
constexpr float PM_LOWEST = -3.4028234e38f;  // a row's maximum before any score: scores of minus infinity have weight 0 whatever stands in front of them

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    mma_bf16(c, a, b0, b1);
  else
    mma16816(c, a, b0, b1);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (!BF16) return half2_bits(a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (!BF16) return h2_to_f2(w);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// (a, b) as TERMS 16-bit values each, the largest first, every one the rounded rest.
template <bool BF16, int TERMS>
__device__ __forceinline__ void split(float a, float b, uint32_t (&w)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    w[i] = pack2<BF16>(a, b);
    if (i + 1 < TERMS) {
      const float2 f = unpack2<BF16>(w[i]);
      a -= f.x;
      b -= f.y;
    }
  }
}
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {  // 16-byte boundaries and sizes
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bar_math() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// What a CTA works on at a time: key tiles t0 .. t1 - 1 (absolute, of 64 keys) of 16 MT rows from R0 on of KV head g of sequence b.
struct Segment {
  uint32_t b, g, R0, t0, t1;
  uint32_t R1;         // rows of the sequence and group end here
  PagedSeq s;
  bool first, last;    // covers the first / the last tile of the block's list
  uint64_t begin, end; // the block's list in the order of all tiles
};

template <int SD, bool BF16, bool F32, int MT>
struct PmShape {
  static constexpr int TERMS = F32 ? (BF16 ? 3 : 2) : 1;
  static constexpr int STAGES = 3;
  static constexpr uint32_t DH = SD * 64, ROWS = 16 * MT;
  static constexpr uint32_t TILE = PM_KEYS * DH * 2;                 // bytes of a tile of keys, or values
  static constexpr uint32_t QP = DH * 2 + 16, PP = PM_KEYS * 2 + 16;  // bytes from a row to the next (16 more: ldmatrix rows in different banks)
  static constexpr uint32_t Q = MT > 1 ? TERMS * ROWS * QP : 0, P = TERMS * ROWS * PP;
  static constexpr uint32_t RAW = DH * (F32 ? 4 : 2) + 16, QR = MT > 1 ? 0 : ROWS * RAW;  // queries as they come (one row block): by bulk copies, a block ahead
  static constexpr uint32_t RING = STAGES * 2 * TILE;
  static constexpr uint32_t MAXIMA = PM_WARPS * ROWS * 4;
  static constexpr size_t bytes(uint32_t batch) { return 1024 + RING + Q + QR + P + 2 * MAXIMA + ROWS * 4 + (size_t)batch * 24 + 8 + (2 * STAGES + 1) * 8 + 16; }
};

template <bool BF16>
constexpr float PM_GAIN = BF16 ? 1.f : 32768.f;  // of probabilities; the largest, 2^15, and its sums with values fit

// Tiles of a sequence's lists (all row blocks alike: those in front of a block's window or behind its last row are passed over), its blocks.
__device__ __forceinline__ void seq_tiles(const PagedSeq &s, uint32_t group, uint32_t rows, uint32_t window, uint32_t &tile0, uint32_t &tiles, uint32_t &blocks) {
  blocks = (s.rows * group + rows - 1) / rows;
  const int lowest = window ? s.pos0 - (int)window + 1 : 0;
  tile0 = lowest > 0 ? (uint32_t)lowest / PM_KEYS : 0;
  const int end = min((int)s.len, s.pos0 + (int)s.rows);  // behind the last row's position
  const uint32_t tile1 = end > 0 ? ((uint32_t)end + PM_KEYS - 1) / PM_KEYS : 0;
  tiles = tile1 > tile0 ? tile1 - tile0 : 1;  // a list is never empty: its rows are written by whoever has it
}

template <int SD, bool BF16, bool F32, int MT>
__global__ void __launch_bounds__(PM_THREADS, MT == 1 ? 2 : 1) paged_mma_kernel(const __grid_constant__ PagedAttnArgs w) {
  using Z = PmShape<SD, BF16, F32, MT>;
  constexpr int TERMS = Z::TERMS, STAGES = Z::STAGES;
  constexpr uint32_t DH = Z::DH, ROWS = Z::ROWS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = reinterpret_cast<uint8_t *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);  // [stage][keys, values][slab][64 rows of 128 bytes, swizzled]
  uint8_t *qs = ring + Z::RING, *qr = qs + Z::Q, *ps = qr + Z::QR;
  float *maxima = reinterpret_cast<float *>(ps + Z::P);        // [warp][row]
  float *sums = maxima + PM_WARPS * ROWS;                      // [warp][row]
  float *factor = sums + PM_WARPS * ROWS;                      // [row]: what scores are multiplied by
  PagedSeq *seqs = reinterpret_cast<PagedSeq *>(factor + ROWS);
  uint64_t *prefix = reinterpret_cast<uint64_t *>(seqs + w.r.batch);  // tiles in front of sequence b
  uint64_t *full = prefix + w.r.batch + 1, *empty = full + STAGES, *qread = empty + STAGES;
  uint32_t *words = reinterpret_cast<uint32_t *>(qread + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(words);
  const uint32_t tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, (int)tid >> 5, 0);
  const uint32_t max_len = w.c.ld_table * w.c.page, group = w.group;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], PM_WARPS);
    }
    mbar_init(qread, PM_WARPS);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w.k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w.v) : "memory");
  }
  pdl_launch_dependents();
  pdl_wait();
  // ---- every CTA's share of the tiles: a list of tiles per row block and KV head, PM_LIST places of its own in front of each
  for (uint32_t b = tid; b < w.r.batch; b += PM_THREADS) {
    const PagedSeq s = seqs[b] = paged_seq(w.r, max_len, b);
    uint32_t tile0, tiles, blocks;
    seq_tiles(s, group, ROWS, w.window, tile0, tiles, blocks);
    prefix[b + 1] = (uint64_t)blocks * w.c.kv_heads * (tiles + PM_LIST);
  }
  __syncthreads();
  if (warp == 0) {
    uint64_t sum = 0;
    for (uint32_t b0 = 0; b0 < w.r.batch; b0 += 32) {
      uint64_t v = b0 + lane < w.r.batch ? prefix[b0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= (uint32_t)o) v += x;
      }
      if (b0 + lane < w.r.batch) prefix[b0 + lane + 1] = sum + v;
      sum += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) prefix[0] = 0;
  }
  __syncthreads();
  const uint64_t total = prefix[w.r.batch], share = (total + gridDim.x - 1) / gridDim.x;
  uint64_t at = min(total, share * blockIdx.x);
  const uint64_t stop = min(total, at + share);

  // The next segment from place `at` on, false when the share ends; lists are [sequence][block][KV head][list's places].
  uint32_t cur = 0;
  auto segment = [&](Segment &g) {
    while (at < stop) {
      if (prefix[cur + 1] <= at) {  // rarely further than the next sequence, but at the share's beginning
        uint32_t lo = cur + 1, hi = w.r.batch;
        if (prefix[lo + 1] <= at) {  // prefix[lo] <= at < prefix[hi]
          while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (prefix[mid] <= at)
              lo = mid;
            else
              hi = mid;
          }
        }
        cur = lo;
      }
      g.b = cur;
      g.s = seqs[cur];
      uint32_t tile0, tiles, blocks;
      seq_tiles(g.s, group, ROWS, w.window, tile0, tiles, blocks);
      const uint32_t places = tiles + PM_LIST;
      const uint64_t in = at - prefix[cur], item = in >> 32 ? in / places : (uint32_t)in / places;
      const uint32_t p = (uint32_t)(in - item * places), n = (uint32_t)min((uint64_t)(places - p), stop - at);
      g.g = (uint32_t)(item % w.c.kv_heads);
      g.R0 = (uint32_t)(item / w.c.kv_heads) * ROWS;
      g.R1 = g.s.rows * group;
      g.begin = at - p + PM_LIST;
      g.end = g.begin + tiles;
      at += n;
      const uint32_t t = max(p, PM_LIST) - PM_LIST, z = max(p + n, PM_LIST) - PM_LIST;
      if (t == z) continue;
      g.first = t == 0;
      g.last = z == tiles;
      // of these, the tiles that some row of the block sees
      const int from = w.window ? g.s.pos0 + (int)(g.R0 / group) - (int)w.window + 1 : 0;
      const int to = g.s.pos0 + (int)((min(g.R1, g.R0 + ROWS) - 1) / group) + 1;  // behind its last row's position
      const uint32_t k0 = from > 0 ? (uint32_t)from / PM_KEYS : 0, k1 = to > 0 ? ((uint32_t)to + PM_KEYS - 1) / PM_KEYS : 0;
      g.t0 = max(k0, tile0 + t);
      g.t1 = max(g.t0, min(k1, tile0 + z));
      return true;
    }
    return false;
  };

  if (warp == PM_WARPS) {
    // ---- pages into the ring.  A tile is 64 / page boxes (or a part of one page) per 64 elements and pool, one lane each.
    const uint32_t box = min(w.c.page, PM_KEYS), boxes = PM_KEYS / box;
    uint32_t it = 0, lists = 0;
    bool ok = true;
    Segment g, n;
    auto page_of = [&](const Segment &x, uint32_t t) {
      const uint32_t p = t * PM_KEYS + lane * box;
      return lane < boxes && t < x.t1 && p < x.s.len ? __ldcg(w.c.table + (size_t)x.b * w.c.ld_table + p / w.c.page) : -1;
    };
    bool more = segment(n);
    int next = more ? page_of(n, n.t0) : -1;
    while (more) {
      g = n;
      const uint32_t rows = min(ROWS, g.R1 - g.R0), row_bytes = w.c.dim * (F32 ? 4 : 2);
      if (g.t0 == g.t1) {
        if ((more = segment(n))) next = page_of(n, n.t0);
        continue;
      }
      for (uint32_t t = g.t0; t < g.t1; ++t, ++it) {
        const int id = next;  // page ids are asked for a tile ahead
        if (t + 1 < g.t1)
          next = page_of(g, t + 1);
        else if ((more = segment(n)))
          next = page_of(n, n.t0);
        const uint32_t st = it % STAGES;
        if (ok) ok = mbar_wait_now(&empty[st], ((it / STAGES) & 1) ^ 1, abort_flag, 800 + st);
        const bool queries = MT == 1 && t == g.t0;  // with the block's first tile
        if (queries) {
          if (ok) ok = mbar_wait_now(qread, (lists & 1) ^ 1, abort_flag, 805);
          ++lists;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (lane == 0 && ok) mbar_arrive_expect_tx(&full[st], 2 * Z::TILE + (queries ? rows * row_bytes : 0));
        __syncwarp();
        if (ok && queries && lane < rows) {
          const uint32_t R = g.R0 + lane;
          const size_t i = (size_t)(g.s.first + R / group) * w.ld_q + (size_t)(g.g * group + R % group) * w.c.dim;
          bulk_load(qr + lane * Z::RAW, static_cast<const uint8_t *>(w.q) + i * (F32 ? 4 : 2), row_bytes, &full[st]);
        }
        if (ok && lane < boxes) {
          const uint32_t p = t * PM_KEYS + lane * box;
          // no page: rows in front of the pool, which read as zeros
          const int row = (uint32_t)id < w.c.pages ? (int)(((uint32_t)id * w.c.kv_heads + g.g) * w.c.page + p % w.c.page) : -(int)PM_KEYS;
          uint8_t *dst = ring + (size_t)st * 2 * Z::TILE + lane * box * 128;
          for (uint32_t c = 0; c < SD; ++c) {
            tma_load_2d(dst + c * PM_KEYS * 128, &w.k, (int)(c * 64), row, &full[st]);
            tma_load_2d(dst + Z::TILE + c * PM_KEYS * 128, &w.v, (int)(c * 64), row, &full[st]);
          }
        }
        __syncwarp();
      }
    }
    if (lane == 0 && *abort_flag) drain_copies(full, it, STAGES);
  } else {
    const uint32_t gq = lane >> 2, t4 = lane & 3, mat = lane >> 3, r8 = lane & 7;
    uint32_t it = 0;
    bool ok = true;
    Segment g;
    while (segment(g)) {
      const uint32_t rows = min(ROWS, g.R1 - g.R0);
      // ---- queries: 16 MT rows, absent ones and elements behind dim as zeros
      uint32_t qf[MT == 1 ? DH / 16 : 1][TERMS][4];
      float rowf[MT][2];
      auto q_at = [&](uint32_t r, uint32_t e) -> float2 {  // elements e, e + 1 (e even) of row r of the block
        if (r >= rows || e >= w.c.dim) return make_float2(0.f, 0.f);
        const uint32_t R = g.R0 + r;
        const size_t i = (size_t)(g.s.first + R / group) * w.ld_q + (size_t)(g.g * group + R % group) * w.c.dim + e;
        if (F32) return __ldcg(reinterpret_cast<const float2 *>(static_cast<const float *>(w.q) + i));
        return unpack2<BF16>(__ldcg(reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(w.q) + i)));
      };
      // fp32 rows are divided by the power of two in front of their largest element, whatever it is, so that their terms keep their bits; in fp16, whose steps end at 2^-24, they
      // are brought to 2^14, and elements down to 2^-17 of the largest keep 22 bits.  The factor itself stays between 2^-126 and 2^127.
      auto down = [&](float most) {
        return most > 0.f && most < INFINITY ? BF16 ? exp2f(-(float)max(-126, min(126, ilogbf(most)))) : exp2f(14.f - (float)max(-113, ilogbf(most))) : 1.f;
      };
      if (MT == 1 && g.t0 < g.t1) {
        if (ok) ok = mbar_wait_now(&full[it % STAGES], (it / STAGES) & 1, abort_flag, 815);
        ok = __all_sync(0xffffffffu, ok);
        auto raw_at = [&](uint32_t r, uint32_t e) -> float2 {
          if (r >= rows || e >= w.c.dim) return make_float2(0.f, 0.f);
          if (F32) return *reinterpret_cast<const float2 *>(qr + r * Z::RAW + e * 4);
          return unpack2<BF16>(*reinterpret_cast<const uint32_t *>(qr + r * Z::RAW + e * 2));
        };
        float2 x[DH / 16][4];
        float most[2] = {0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            x[ks][c] = raw_at(gq + (c & 1) * 8, ks * 16 + (c >> 1) * 8 + 2 * t4);
            most[c & 1] = fmaxf(most[c & 1], fmaxf(fabsf(x[ks][c].x), fabsf(x[ks][c].y)));
          }
        float f[2] = {1.f, 1.f};
        if (F32) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            most[c] = fmaxf(most[c], __shfl_xor_sync(0xffffffffu, most[c], 1));
            most[c] = fmaxf(most[c], __shfl_xor_sync(0xffffffffu, most[c], 2));
            f[c] = down(most[c]);
          }
        }
        rowf[0][0] = w.scale2 / f[0];
        rowf[0][1] = w.scale2 / f[1];
#pragma unroll
        for (int ks = 0; ks < DH / 16; ++ks)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t v[TERMS];
            split<BF16, TERMS>(x[ks][c].x * f[c & 1], x[ks][c].y * f[c & 1], v);
#pragma unroll
            for (int i = 0; i < TERMS; ++i) qf[ks][i][c] = v[i];
          }
        __syncwarp();
        if (lane == 0) mbar_arrive(qread);
      } else {
        bar_math();  // the rows before have been read, and their sums: a segment of no tile writes its own with no other barrier in front
      }
      if (MT > 1) {
        for (uint32_t r = warp; r < ROWS; r += PM_WARPS) {
          float2 x[DH / 64];
          float most = 0.f;
#pragma unroll
          for (int e = 0; e < DH / 64; ++e) {
            x[e] = q_at(r, e * 64 + 2 * lane);
            most = fmaxf(most, fmaxf(fabsf(x[e].x), fabsf(x[e].y)));
          }
          const float f = F32 ? down(warp_max(most)) : 1.f;
          if (lane == 0) factor[r] = w.scale2 / f;
#pragma unroll
          for (int e = 0; e < DH / 64; ++e) {
            uint32_t v[TERMS];
            split<BF16, TERMS>(x[e].x * f, x[e].y * f, v);
#pragma unroll
            for (int i = 0; i < TERMS; ++i) *reinterpret_cast<uint32_t *>(qs + (size_t)(i * ROWS + r) * Z::QP + e * 128 + lane * 4) = v[i];
          }
        }
        bar_math();
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          rowf[m][0] = factor[m * 16 + gq];
          rowf[m][1] = factor[m * 16 + gq + 8];
        }
      }
      // Keys that the thread's rows see: lim0 <= key < lim1.
      int lim0[MT][2], lim1[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t r = m * 16 + gq + c * 8;
          const int pos = g.s.pos0 + (int)((g.R0 + r) / group);
          lim1[m][c] = r < rows ? pos + 1 : 0;
          lim0[m][c] = w.window && pos >= (int)w.window ? pos - (int)w.window + 1 : 0;
        }
      // Tiles that every row sees whole need no masks.
      const int pos_lo = g.s.pos0 + (int)(g.R0 / group), pos_hi = g.s.pos0 + (int)((g.R0 + rows - 1) / group);
      const int whole0 = w.window ? max(0, pos_hi - (int)w.window + 1) : 0, whole1 = pos_lo + 1;
      float mx[MT][2], l[MT][2], o[MT][DH / 32][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        mx[m][0] = mx[m][1] = PM_LOWEST;
        l[m][0] = l[m][1] = 0.f;
#pragma unroll
        for (int n = 0; n < DH / 32; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[m][n][j] = 0.f;
      }
      for (uint32_t t = g.t0; t < g.t1; ++t, ++it) {
        const uint32_t st = it % STAGES;
        uint8_t *kt = ring + (size_t)st * 2 * Z::TILE, *vt = kt + Z::TILE;
        if (ok) ok = mbar_wait_now(&full[st], (it / STAGES) & 1, abort_flag, 810 + st);
        ok = __all_sync(0xffffffffu, ok);
        // ---- scores of the warp's 16 keys.  The tensor core cuts sums off at the accumulator's last bit, the further the more is in it: fp32 calls add two steps of 16 elements at a time to the
        // score by an fp32 add that rounds (error of one sequence of 577 5.6e-7 -> 2.8e-7, of 16 around 4096 7.3e-7 -> 3.3e-7, the plain form's 2.2e-7 and 5.9e-7; 13.05 -> 13.15 and
        // 59.6 -> 60.3 us, 512 rows of 4096 827 -> 883.  One step at a time: 2.5e-7 and 3.0e-7, 61.1 us.)
        constexpr int TOGETHER = 2;
        float s[MT][2][4], sum[MT][2][4] = {};
        auto add = [&] {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                sum[m][n][j] += s[m][n][j];
                s[m][n][j] = 0.f;
              }
        };
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[m][n][j] = 0.f;
        const uint32_t key = warp * 16 + (mat >> 1) * 8 + r8;  // the row whose address this lane gives to ldmatrix
#pragma unroll
        for (int ks = 0; ks < (int)DH / 16; ++ks) {
          uint32_t kb[4];
          if (F32 && ks && ks % TOGETHER == 0) add();
          ldsm_x4(kb, kt + (ks / 4) * PM_KEYS * 128 + key * 128 + ((((ks & 3) * 2 + (mat & 1)) ^ (key & 7)) << 4));
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = TERMS - 1; i >= 0; --i) {
              uint32_t a[4];
              if (MT == 1) {
#pragma unroll
                for (int c = 0; c < 4; ++c) a[c] = qf[ks][i][c];
              } else {
                ldsm_x4(a, qs + (size_t)(i * ROWS + m * 16 + (mat & 1) * 8 + r8) * Z::QP + ks * 32 + (mat >> 1) * 16);
              }
              mma<BF16>(s[m][0], a, kb[0], kb[1]);
              mma<BF16>(s[m][1], a, kb[2], kb[3]);
            }
        }
        const int k0 = (int)(t * PM_KEYS);
        const bool masks = k0 < whole0 || k0 > whole1 - (int)PM_KEYS;  // no sum with k0: positions end at 2^31
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float tm[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float x = (F32 ? s[m][n][j] + sum[m][n][j] : s[m][n][j]) * rowf[m][j >> 1];
              if (masks) {
                const int k = k0 + warp * 16 + n * 8 + (int)(2 * t4) + (j & 1);
                if (k < lim0[m][j >> 1] || k >= lim1[m][j >> 1]) x = -INFINITY;
              }
              s[m][n][j] = x;
              tm[j >> 1] = fmaxf(tm[j >> 1], x);
            }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            tm[c] = fmaxf(tm[c], __shfl_xor_sync(0xffffffffu, tm[c], 1));
            tm[c] = fmaxf(tm[c], __shfl_xor_sync(0xffffffffu, tm[c], 2));
            if (t4 == 0) maxima[warp * ROWS + m * 16 + gq + c * 8] = tm[c];
          }
        }
        // ---- values behind the sequence's end are whatever the page held before: zeros
        const int end = min((int)g.s.len, g.s.pos0 + (int)g.s.rows);
        if (k0 > end - (int)PM_KEYS) {
          const uint32_t from = (uint32_t)max(0, end - k0);
          for (uint32_t i = tid; i < (PM_KEYS - from) * SD * 8; i += 32 * PM_WARPS) {
            const uint32_t c = i / ((PM_KEYS - from) * 8), j = i % ((PM_KEYS - from) * 8);
            *reinterpret_cast<uint4 *>(vt + c * PM_KEYS * 128 + from * 128 + j * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        bar_math();
        // ---- probabilities
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t r = m * 16 + gq + c * 8;
            float nm = mx[m][c];
#pragma unroll
            for (int x = 0; x < (int)PM_WARPS; ++x) nm = fmaxf(nm, maxima[x * ROWS + r]);
            const float f = ex2(mx[m][c] - nm);
            mx[m][c] = nm;
            l[m][c] *= f;
#pragma unroll
            for (int n = 0; n < (int)DH / 32; ++n) {
              o[m][n][2 * c] *= f;
              o[m][n][2 * c + 1] *= f;
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const float p0 = PM_GAIN<BF16> * ex2(s[m][n][2 * c] - nm), p1 = PM_GAIN<BF16> * ex2(s[m][n][2 * c + 1] - nm);
              l[m][c] += p0 + p1;
              uint32_t v[TERMS];
              split<BF16, TERMS>(p0, p1, v);
#pragma unroll
              for (int i = 0; i < TERMS; ++i) *reinterpret_cast<uint32_t *>(ps + (size_t)(i * ROWS + r) * Z::PP + (warp * 16 + n * 8 + 2 * t4) * 2) = v[i];
            }
          }
        }
        bar_math();
        // ---- outputs: the warp's DH / 4 elements, 64 keys.  The tensor core cuts sums off at the accumulator's last bit: a tile's products meet in
        // accumulators of their own, added to the row's by an fp32 add that rounds (error of 16 sequences over 4096 keys, fp32: 7.2e-7; without 4.0e-6).
        float po[MT][DH / 32][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < (int)DH / 32; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) po[m][n][j] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t vb[DH / 64][4];
          const uint32_t vk = kk * 16 + (mat & 1) * 8 + r8;
#pragma unroll
          for (int n = 0; n < (int)DH / 64; ++n) {
            const uint32_t e = warp * (DH / 4) + n * 16 + (mat >> 1) * 8;
            ldsm_x4_trans(vb[n], vt + (e / 64) * PM_KEYS * 128 + vk * 128 + (((e % 64 / 8) ^ (vk & 7)) << 4));
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = TERMS - 1; i >= 0; --i) {
              uint32_t a[4];
              ldsm_x4(a, ps + (size_t)(i * ROWS + m * 16 + (mat & 1) * 8 + r8) * Z::PP + kk * 32 + (mat >> 1) * 16);
#pragma unroll
              for (int n = 0; n < (int)DH / 64; ++n) {
                mma<BF16>(po[m][2 * n], a, vb[n][0], vb[n][1]);
                mma<BF16>(po[m][2 * n + 1], a, vb[n][2], vb[n][3]);
              }
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < (int)DH / 32; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[m][n][j] += po[m][n][j];
        if (k0 > end - (int)PM_KEYS) fence_proxy_async();  // the zeros are in front of the next copy
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }
      // ---- sums of the warps' keys
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = l[m][c];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if (t4 == 0) sums[warp * ROWS + m * 16 + gq + c * 8] = x;
        }
      bar_math();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t r = m * 16 + gq + c * 8;
          l[m][c] = (sums[r] + sums[ROWS + r]) + (sums[2 * ROWS + r] + sums[3 * ROWS + r]);
        }
      // ---- values of hidden keys that are no finite numbers (0 times such a value is none): the row's elements again, over the keys it sees
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t r = m * 16 + gq + c * 8;
          float z = 0.f;  // 0, or NaN
#pragma unroll
          for (int n = 0; n < (int)DH / 16; ++n) z = fmaf(o[m][n / 2][2 * c + (n & 1)], 0.f, z);
          if (z != 0.f && r < rows && isfinite(l[m][c])) {
            float y[DH / 16];
#pragma unroll
            for (int n = 0; n < (int)DH / 16; ++n) y[n] = o[m][n / 2][2 * c + (n & 1)];
            paged_again<DH / 16>(w, BF16, F32, g.b, g.s, g.g, g.R0 + r, [&](int n) { return warp * (DH / 4) + n / 2 * 8 + 2 * t4 + (n & 1); },
                                 max(lim0[m][c], (int)(g.t0 * PM_KEYS)), min(lim1[m][c], (int)min(g.t1 * PM_KEYS, 0x7fffffffu)), mx[m][c], PM_GAIN<BF16>, y);
#pragma unroll
            for (int n = 0; n < (int)DH / 16; ++n) o[m][n / 2][2 * c + (n & 1)] = y[n];
          }
        }
      // ---- a part of the block's tiles: to the workspace, and whoever is last joins the parts
      bool mine = true;
      if (!(g.first && g.last)) {
        const uint32_t c0 = (uint32_t)(g.begin / share), c1 = (uint32_t)((g.end - 1) / share);
        auto part = [&](uint32_t cta) {  // a CTA has at most one part that is no beginning of a list, and one that is
          return w.parts + (size_t)(2 * cta + (cta == c0 ? 1 : 0)) * PAGED_MMA_PART;
        };
        float *p = part(blockIdx.x);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t r = m * 16 + gq + c * 8;
            if (r >= rows) continue;
            if (t4 == 0 && warp == 0) {
              __stcg(p + r * 2, mx[m][c]);
              __stcg(p + r * 2 + 1, l[m][c]);
            }
#pragma unroll
            for (int n = 0; n < (int)DH / 32; ++n)
              __stcg(reinterpret_cast<float2 *>(p + 2 * ROWS + r * DH + warp * (DH / 4) + n * 8 + 2 * t4), make_float2(o[m][n][2 * c], o[m][n][2 * c + 1]));
          }
        __threadfence();
        bar_math();
        if (tid == 0) {
          const uint32_t before = atomicAdd(w.tickets + c0, 1u);
          if (before == c1 - c0) w.tickets[c0] = 0;  // all are here: the ticket is free again
          words[1] = before;
          __threadfence();
        }
        bar_math();
        mine = words[1] == c1 - c0;
        if (mine) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t r = m * 16 + gq + c * 8;
              float big = PM_LOWEST;
              if (r < rows)
                for (uint32_t x = c0; x <= c1; ++x) big = fmaxf(big, __ldcg(part(x) + r * 2));
              mx[m][c] = big;
              l[m][c] = 0.f;
#pragma unroll
              for (int n = 0; n < (int)DH / 32; ++n) o[m][n][2 * c] = o[m][n][2 * c + 1] = 0.f;
              if (r < rows)
                for (uint32_t x = c0; x <= c1; ++x) {
                  const float *y = part(x);
                  const float f = ex2(__ldcg(y + r * 2) - big);
                  l[m][c] = fmaf(__ldcg(y + r * 2 + 1), f, l[m][c]);
#pragma unroll
                  for (int n = 0; n < (int)DH / 32; ++n) {
                    const float2 z = __ldcg(reinterpret_cast<const float2 *>(y + 2 * ROWS + r * DH + warp * (DH / 4) + n * 8 + 2 * t4));
                    o[m][n][2 * c] = fmaf(z.x, f, o[m][n][2 * c]);
                    o[m][n][2 * c + 1] = fmaf(z.y, f, o[m][n][2 * c + 1]);
                  }
                }
            }
        }
      }
      if (mine && ok) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t r = m * 16 + gq + c * 8, R = g.R0 + r;
            if (r >= rows) continue;
            const float inv = l[m][c] == 0.f ? 0.f : 1.f / l[m][c];
            const size_t i = (size_t)(g.s.first + R / group) * w.ld_o + (size_t)(g.g * group + R % group) * w.c.dim;
#pragma unroll
            for (int n = 0; n < (int)DH / 32; ++n) {
              const uint32_t e = warp * (DH / 4) + n * 8 + 2 * t4;
              if (e >= w.c.dim) continue;
              const float x = o[m][n][2 * c] * inv, y = o[m][n][2 * c + 1] * inv;
              if (F32)
                *reinterpret_cast<float2 *>(static_cast<float *>(w.o) + i + e) = make_float2(x, y);
              else
                *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(w.o) + i + e) = pack2<BF16>(x, y);
            }
          }
      }
    }
  }
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicCAS(w.error, 0, *abort_flag);
}

template <int SD, bool BF16, bool F32, int MT>
int launch_mma(cudaStream_t stream, const PagedAttnArgs &w) {
  using Z = PmShape<SD, BF16, F32, MT>;
  const size_t smem = Z::bytes(w.r.batch);
  // A CTA's memory grows with the batch (24 bytes a sequence): the most sequences with which an SM holds two.
  static int two[64] = {};  // 1 + that
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  if (two[dev] == 0) {
    GRETA_CUDA_TRY(cudaFuncSetAttribute(paged_mma_kernel<SD, BF16, F32, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Z::bytes(PAGED_MAX_BATCH)));
    int most = 0;
    for (int step = (int)PAGED_MAX_BATCH; step; step /= 2) {
      int n = 0;
      if (most + step <= (int)PAGED_MAX_BATCH)
        GRETA_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, paged_mma_kernel<SD, BF16, F32, MT>, PM_THREADS, Z::bytes(most + step)));
      if (n >= (int)PAGED_CTAS_PER_SM) most += step;
    }
    two[dev] = most + 1;
  }
  const uint32_t grid = std::min<uint32_t>(PAGED_MAX_CTAS, ((int)w.r.batch < two[dev] ? PAGED_CTAS_PER_SM : 1) * (uint32_t)sm_count());
  GRETA_CUDA_TRY(launch_pdl(paged_mma_kernel<SD, BF16, F32, MT>, dim3(grid), dim3(PM_THREADS), smem, stream, w));
  return launched("paged_mma_kernel");
}

template <int SD, bool BF16>
int launch_mma(cudaStream_t stream, const PagedAttnArgs &w, bool f32, bool many) {
  if (f32) return many ? launch_mma<SD, BF16, true, 4>(stream, w) : launch_mma<SD, BF16, true, 1>(stream, w);
  return many ? launch_mma<SD, BF16, false, 4>(stream, w) : launch_mma<SD, BF16, false, 1>(stream, w);
}

}  // namespace


namespace {

// A pool as rows of `dim` elements, boxes of `rows` rows of 64 elements; what lies outside (rows in front of the pool, elements behind dim) reads as zeros.
int pool_map(CUtensorMap *map, EncodeTiledFn enc, const greta_paged_cache &c, void *pool, uint32_t rows) {
  const cuuint64_t dims[2] = {c.dim, (cuuint64_t)c.pages * c.kv_heads * c.page}, strides[1] = {(cuuint64_t)c.dim * 2};
  const cuuint32_t box[2] = {64, rows}, one[2] = {1, 1};
  const CUresult r = enc(map, c.fmt == GRETA_FMT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, pool, dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return GRETA_OK;
  set_error("paged_attn: cuTensorMapEncodeTiled failed with code %d", (int)r);
  return GRETA_ERR_INVALID_ARGS;
}

}  // namespace

extern "C" {

size_t greta_cuda_paged_attn_workspace_bytes(uint32_t dim) {
  (void)dim;
  return PAGED_TICKETS + PAGED_PARTS * 4;
}

int greta_cuda_paged_attn(greta_stream_t stream, const greta_paged_cache *cache, const greta_ragged *rows, const void *q, int q_fmt, uint32_t ld_q, void *o,
                          uint32_t ld_o, uint32_t heads, float scale, uint32_t window, void *workspace, size_t workspace_bytes) {
  if (int rc = paged_check(cache, rows, "paged_attn")) return rc;
  const uint32_t d = cache->dim;
  GRETA_REQUIRE(q && o && workspace, "paged_attn: null pointer");
  GRETA_REQUIRE(q_fmt == GRETA_FMT_F32 || q_fmt == cache->fmt, "paged_attn: queries of format %d over a cache of format %d", q_fmt, cache->fmt);
  GRETA_REQUIRE(heads >= 1 && heads <= 65535 && heads % cache->kv_heads == 0, "paged_attn: %u heads over %u", heads, cache->kv_heads);
  GRETA_REQUIRE(ld_q >= heads * d && ld_o >= heads * d, "paged_attn: rows closer than their elements");
  GRETA_REQUIRE(aligned16(q) && aligned16(o) && (size_t)ld_q * paged_size(q_fmt) % 16 == 0 && (size_t)ld_o * paged_size(q_fmt) % 16 == 0,
                "paged_attn: rows that do not begin at 16-byte boundaries");
  GRETA_REQUIRE(q != o, "paged_attn: in place");
  const float scale2 = scale * 1.4426950408889634f;  // of powers of two
  GRETA_REQUIRE(window < (1u << 31) && scale2 > 0 && isfinite(scale2), "paged_attn: window %u, scale %g", window, scale);
  GRETA_REQUIRE(aligned16(workspace) && workspace_bytes >= greta_cuda_paged_attn_workspace_bytes(d), "paged_attn: workspace of %zu bytes, %zu needed", workspace_bytes,
                greta_cuda_paged_attn_workspace_bytes(d));
  const size_t row = (size_t)heads * d * paged_size(q_fmt);
  GRETA_REQUIRE(!rows_meet(q, (size_t)ld_q * paged_size(q_fmt), row, o, (size_t)ld_o * paged_size(q_fmt), row, rows->tokens), "paged_attn: o overlaps q");
  if (rows->tokens == 0) return GRETA_OK;
  EncodeTiledFn enc = encode_tiled();
  if (!enc) {
    set_error("paged_attn: cuTensorMapEncodeTiled is not available from this driver");
    return GRETA_ERR_NOT_IMPLEMENTED;
  }
  PagedAttnArgs w{};
  w.c = *cache;
  w.r = *rows;
  w.q = q;
  w.o = o;
  w.ld_q = ld_q;
  w.ld_o = ld_o;
  w.group = heads / cache->kv_heads;
  w.window = window;
  w.scale2 = scale2;
  w.tickets = static_cast<uint32_t *>(workspace);
  w.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + PAGED_TICKETS);
  if (int rc = gemm_ts_error_word(&w.error)) return rc;
  const uint32_t most = rows->max_rows ? std::min(rows->max_rows, rows->tokens) : rows->tokens;
  const bool many = (uint64_t)most * w.group > 16, bf16 = cache->fmt == GRETA_FMT_BF16, f32 = q_fmt == GRETA_FMT_F32;
  // More than 16 rows of 16 bits: the form for portions, whose blocks of 256 rows are mostly empty then, but whose tensor core does not wait for operands.  Eight sequences of five
  // rows of 8 heads: 18.6 us, 28 here; of three: 18.2 and 23.8; 16 of one row of 32 heads over 4096 keys: 28 and 43; 24 of 16 rows over up to 6000: 78 and 411.
  const bool tc = many && !f32 && paged_tc_fits(w);
  const uint32_t box = std::min(cache->page, tc ? 128 : PM_KEYS);
  if (int rc = pool_map(&w.k, enc, *cache, cache->k, box)) return rc;
  if (int rc = pool_map(&w.v, enc, *cache, cache->v, box)) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tc) return paged_attn_tc(s, w, heads);
  if (d > 64) return bf16 ? launch_mma<2, true>(s, w, f32, many) : launch_mma<2, false>(s, w, f32, many);
  return bf16 ? launch_mma<1, true>(s, w, f32, many) : launch_mma<1, false>(s, w, f32, many);
}

}  // extern "C"
