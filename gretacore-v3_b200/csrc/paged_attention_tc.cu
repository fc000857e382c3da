// Attention of a ragged batch's new rows over a paged cache on the 5th-generation tensor cores: portions of prompts, queries of the cache's type.
//
// A CTA takes a block of 256 query rows of one KV head as two tiles of 128: row R of a sequence and KV head is token R / group, head R % group, so a tile
// is 128 / group tokens with all their heads and every key tile is fetched once for them.  Keys come in tiles of 128, page by page, by TMA (a page's rows of a head
// are contiguous); queries by TMA as boxes of [tokens][group][64].
//   warp 0: copies; warp 1: MMAs; warps 2-9 and 10-17: the rows of the first and
//   second tile, two threads each (64 keys of a tile, half of the outputs): maxima, probabilities, outputs.
// The two tiles take turns: while the tensor core multiplies one (P V of this key tile, Q K of the next), the other's probabilities are made.
//   tensor memory: scores of tile A and B at columns 0 and 128, each half of which is overwritten by its probabilities (32 columns), outputs at 256 and 384.
// A row's sums are rescaled only when its maximum has grown by more than 2^8; the scores' barrier of a key tile says that
// the products of the one before are in, so the rows' own threads do that.
// Probabilities are rounded to the cache's type for the second product (half a step: 2^-11 or 2^-8 of each); the sum of them is taken in fp32 before that.  fp16's steps end at
// 2^-24, so they are taken against the maximum less 7 there: up to 2^15, sums as well, and the division at the end takes it out.  Weights down to 2^-21 of a row's largest keep their 11 bits
// (4096 keys behind one of no value and a score 14 higher: error 3.5e-4 of the outputs' size, without 3.5e-3).
//
// What bounds it: the tensor core (55 % of the time) and the exponentials (special-function unit 56 %, 16 a cycle and SM in any type) take turns that do not overlap whole; every
// row's 64 scores, bounds and sums take the 96 registers that 18 warps leave a thread (a spill in this loop goes to the second-level cache, since tiles leave the first 28 KB:
// 58 us became 68).  512 rows behind 15872 keys, 64 heads over 8 of 128: 237 us (1150 TFLOP/s), 268 when the power limit has lowered the clocks; a prompt of
// 2048, 32 heads: 44 us; of 8192, clocks lowered: 564 (980 TFLOP/s).
// Blocks: where there are many, whole ones are drawn from a counter, the longest first (no joining); where drawn ones would leave SMs idle longer than joining takes, all
// CTAs get equal shares of the places, and the last of a block's CTAs to finish joins its parts in their order.
#include <math.h>
#include <stddef.h>

#include <algorithm>
#include <type_traits>

#include "mma_device.cuh"
#include "paged_attention.cuh"
#include "tc_device.cuh"

using namespace greta;

namespace {

constexpr uint32_t PT_ROWS = 128, PT_KEYS = 128, PT_THREADS = 576, PT_UNITS = 4, PT_TMEM = 512;
constexpr uint32_t PT_TILE1 = 6, PT_TILE2 = 6, PT_LIST1 = 10, PT_LIST2 = 18;  // places of a key tile and of a block's beginning and end, with one half and with two
constexpr uint32_t PT_JOIN = 32;                                               // what joining the shares' parts costs
constexpr uint32_t PT_MAX_CTAS = PAGED_TC_CTAS;
constexpr uint32_t PT_BARRIERS = 28, PT_SMALL = 3328;  // of a CTA; bytes of shared memory for them, exchanges, segments and words
constexpr uint32_t PT_SLAB = 128 * 128;  // bytes of 64 elements of 128 rows
constexpr float PT_LAZY = 8.f;           // log2 of what a row's maximum may grow by before its sums are rescaled
constexpr float PT_LOWEST = -3.4028234e38f;  // a row's maximum before any score
template <bool BF16>
constexpr float PT_BELOW = BF16 ? 0.f : 7.f;  // m2 is this much (log2) below the maximum that it stands for

__device__ __forceinline__ void tma_load_3d(void *smem_dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(smem_dst)),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
               : "memory");
}
// On the critical path: waits that the hardware ends (a time hint wakes late; testing without rest takes issue slots from the warps that compute).
// Shared memory is addressed with 32 bits: generic pointers take twice the registers, of which a row's scores leave none.
__device__ __forceinline__ uint32_t lds(uint32_t at) {
  uint32_t x;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ void sts(uint32_t at, uint32_t x) { asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(at), "r"(x) : "memory"); }
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool test(uint32_t bar, uint32_t parity) {  // at once
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// No call: what a caller's registers hold would go to local memory around it, and come back from the second-level cache when the wait is over.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t abort_flag, int code) {
  if (try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  bool ok;
  do {
    ok = try_wait(bar, parity);
    if (!ok && clock64() - t0 > WAIT_LIMIT_CYCLES) sts(abort_flag, code);
  } while (!ok && !lds(abort_flag));
  return ok;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (!BF16) return half2_bits(a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
               "r"(r[6]), "r"(r[7])
               : "memory");
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
// A block of rows of one sequence and KV head: its tokens as two halves, and the key tiles lo .. hi - 1 that each sees; t0 .. t1 - 1 is both.
struct Block {
  uint32_t token0, tokens[2], lo[2], hi[2], t0, t1;
};
__device__ __forceinline__ Block block_of(const PagedSeq &s, uint32_t j, uint32_t TT, uint32_t window) {
  Block k;
  k.token0 = j * 2 * TT;
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t first = k.token0 + i * TT;
    k.tokens[i] = first < s.rows ? min(TT, s.rows - first) : 0;
    const int pos = s.pos0 + (int)first, end = pos + (int)k.tokens[i];  // positions pos .. end - 1
    const int from = window ? pos - (int)window + 1 : 0;
    k.lo[i] = k.tokens[i] == 0 ? k.lo[0] : from > 0 ? (uint32_t)from / PT_KEYS : 0;
    k.hi[i] = k.tokens[i] && end > 0 ? ((uint32_t)end + PT_KEYS - 1) / PT_KEYS : k.lo[i];
  }
  // The second half's tiles begin and end no earlier than the first's, and there is none between them: its first row follows the first half's last.
  k.t0 = k.lo[0];
  k.t1 = max(k.hi[0], k.hi[1]);
  return k;
}
// What a block costs, in places of about 0.3 us: a key tile of two halves, or of one (whose tensor core and special-function unit wait for each other), and its beginning
// and end.  The tiles of a block that sees no key are taken for one.
__device__ __forceinline__ uint32_t tile_places(const Block &k) { return k.tokens[1] ? PT_TILE2 : PT_TILE1; }
__device__ __forceinline__ uint32_t list_places(const Block &k) { return k.tokens[1] ? PT_LIST2 : PT_LIST1; }
__device__ __forceinline__ uint32_t places_of(const Block &k) { return max(1u, k.t1 - k.t0) * tile_places(k) + list_places(k); }

// What a CTA works on at a time: a block of a KV head, its tiles clipped to k.t0 .. k.t1 - 1.
struct Segment {
  Block k;
  PagedSeq s;
  uint32_t b, g;
  uint32_t whole, tail;    // all of the block; rows of the last tile that lie behind the sequence's end
  uint32_t c0, c1;         // the CTAs that share the block
  uint32_t clear0[2], clear1[2];  // of a half: the tiles that all its rows see whole
  int pos[2];              // of a half: its first row's position
  uint32_t more;           // 0: there was none
};

// What is to be done, in the order of its places: sequences, their blocks from the last (and longest) to the first, KV heads.  Used by all lanes of a warp.
struct Finder {
  const PagedAttnArgs &w;
  const uint32_t *prefix;  // places (or blocks) in front of a sequence, and of the end
  const PagedSeq *seqs;
  const uint32_t share;    // places of each CTA
  const uint32_t TT, G, lane;
  uint32_t at, stop, begin = 0;  // the next place, the end of the CTA's; the first place of the block that `at` lies in
  uint32_t cur = 0, jj = 0, kvh = 0;  // that block: sequence, number from the last, KV head
  bool found = false;

  __device__ Finder(const PagedAttnArgs &w, const uint32_t *prefix, const PagedSeq *seqs, uint32_t share)
      : w(w), prefix(prefix), seqs(seqs), share(share), TT(PT_ROWS / w.group), G(w.c.kv_heads), lane(threadIdx.x & 31) {
    at = min(prefix[w.r.batch], share * blockIdx.x);
    stop = min(prefix[w.r.batch], at + share);
  }
  __device__ uint32_t blocks_of(const PagedSeq &s) const { return (s.rows + 2 * TT - 1) / (2 * TT); }
  __device__ uint32_t seq_at(uint32_t x) const {  // prefix[b] <= x < prefix[b + 1]
    uint32_t lo = 0, hi = w.r.batch;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (prefix[mid] <= x)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  }
  __device__ void finish(Segment &g) const {
    g.whole = g.c0 == g.c1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int first = g.s.pos0 + (int)(g.k.token0 + i * TT), last = first + (int)g.k.tokens[i] - 1;
      g.pos[i] = first;
      g.clear0[i] = w.window && last >= (int)w.window ? (uint32_t)(last - (int)w.window + PT_KEYS) / PT_KEYS : 0;
      g.clear1[i] = first < 0 ? 0 : (uint32_t)(first + 1) / PT_KEYS;
    }
  }
  __device__ uint32_t tail(const Segment &g) const {
    const uint32_t end = (uint32_t)(g.s.pos0 + (int)g.s.rows), tiles = g.k.t1 * PT_KEYS;  // up to 2^31
    return g.k.t1 > g.k.t0 && tiles > end ? tiles - end : 0;
  }
  // A whole block by its number.
  __device__ void block(uint32_t x, Segment &g) const {
    g.b = seq_at(x);
    g.s = seqs[g.b];
    const uint32_t in = x - prefix[g.b];
    g.g = in % G;
    g.k = block_of(g.s, blocks_of(g.s) - 1 - in / G, TT, w.window);
    g.c0 = g.c1 = 0;
    g.tail = tail(g);
    finish(g);
  }
  __device__ void search() {  // the share's beginning: which sequence, and which of its blocks, 32 at a time
    cur = seq_at(at);
    const PagedSeq s = seqs[cur];
    const uint32_t blocks = blocks_of(s);
    uint32_t before = prefix[cur];
    for (uint32_t j0 = 0; !found; j0 += 32) {
      const uint32_t mine = j0 + lane < blocks ? places_of(block_of(s, blocks - 1 - j0 - lane, TT, w.window)) * G : 0;
      uint32_t v = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, before + v > at);
      found = hit || j0 + 32 >= blocks;
      if (found) {
        const int l = hit ? __ffs(hit) - 1 : 0;
        jj = j0 + l;
        const uint32_t first = __shfl_sync(0xffffffffu, v - mine, l), each = __shfl_sync(0xffffffffu, mine, l) / G;
        kvh = (at - before - first) / each;
        begin = before + first + kvh * each;
      }
      before += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  // The next part of the CTA's share.
  __device__ bool part(Segment &g) {
    while (at < stop) {
      if (!found) search();
      g.b = cur;
      g.g = kvh;
      g.s = seqs[cur];
      const uint32_t blocks = blocks_of(g.s);
      g.k = block_of(g.s, blocks - 1 - jj, TT, w.window);
      const uint32_t tiles = g.k.t1 - g.k.t0, places = places_of(g.k), p = at - begin, n = min(places - p, stop - at);
      // A tile is the CTA's that its first place falls to.
      const uint32_t each = tile_places(g.k), list = list_places(g.k), end = begin + places;
      auto tile_at = [&](uint32_t x) { return x <= list ? 0 : (x - list + each - 1) / each; };
      const uint32_t a = tile_at(p), z = tile_at(p + n), c0 = (begin + list) / share, c1 = (end - each) / share;
      at += n;
      if (at == end) {  // on to the next block
        begin = end;
        if (++kvh == G) {
          kvh = 0;
          if (++jj == blocks) {
            jj = 0;
            while (++cur < w.r.batch && prefix[cur + 1] == prefix[cur]) {
            }
          }
        }
      }
      if (a == z) continue;
      g.c0 = c0;
      g.c1 = c1;
      const uint32_t t0 = g.k.t0 + min(a, tiles), t1 = g.k.t0 + min(z, tiles);
      const bool to_end = t1 == g.k.t1;
      g.k.t0 = t0;
      g.k.t1 = t1;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        g.k.lo[i] = min(max(g.k.lo[i], t0), t1);
        g.k.hi[i] = max(min(g.k.hi[i], t1), g.k.lo[i]);
      }
      g.tail = to_end ? tail(g) : 0;
      finish(g);
      return true;
    }
    return false;
  }
};

template <int SD, bool BF16>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_tc_kernel(const __grid_constant__ PagedAttnArgs w) {
  constexpr uint32_t DH = SD * 64, UNIT = SD * PT_SLAB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *qs = smem, *ring = qs + 2 * UNIT;  // queries of both halves; keys and values in turn
  uint8_t *small = ring + PT_UNITS * UNIT;
  constexpr uint32_t MEET = 0, BARS = 4 * PT_ROWS * 4;  // [half][column half][row] floats that the two threads of a row tell each other (512 bytes apart); barriers
  constexpr uint32_t FULL = BARS / 8, EMPTY = FULL + PT_UNITS, QF = EMPTY + PT_UNITS, QE = QF + 2, SF = QE + 2, PF = SF + 2, FIN = PF + 4, NF = FIN + 2, NE = NF + 2;
  static_assert(NE + 2 <= BARS / 8 + PT_BARRIERS, "barriers");
  uint64_t *all = reinterpret_cast<uint64_t *>(small), *full = all + FULL, *empty = all + EMPTY, *qf = all + QF, *qe = all + QE, *sf = all + SF, *pf = all + PF, *fin = all + FIN;
  uint64_t *nf = all + NF, *ne = all + NE;  // the next segment is there; is done with
  // Behind the barriers: [row] its token and head (divisions by the group, once); two segments (warp 0 finds them, one ahead; the others leave in them what they
  // need late); words; and what depends on the batch.
  constexpr uint32_t ROWS = BARS + PT_BARRIERS * 8, SEGMENTS = ROWS + PT_ROWS * 4, WORDS = SEGMENTS + 2 * sizeof(Segment);
  Segment *segments = reinterpret_cast<Segment *>(small + SEGMENTS);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(small + WORDS), *ticket = tmem_slot + 1, *limits = ticket + 1;  // limits: cost of the largest and of the smallest block
  volatile int *abort_flag = reinterpret_cast<volatile int *>(limits + 2);
  constexpr uint32_t ABORT = WORDS + 16;
  uint32_t *prefix = reinterpret_cast<uint32_t *>(small + PT_SMALL);  // [batch + 1]: places (or blocks) in front of a sequence; and [batch] its blocks
  uint32_t *blocks_in = prefix + w.r.batch + 1;
  PagedSeq *seqs = reinterpret_cast<PagedSeq *>(blocks_in + w.r.batch);
  static_assert(WORDS + 32 <= PT_SMALL, "small things");
  const uint32_t sm = smem_u32(small);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t group = w.group, TT = PT_ROWS / group, G = w.c.kv_heads, N = gridDim.x;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < PT_UNITS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&qf[i], 1);
      mbar_init(&qe[i], 1);
      mbar_init(&sf[i], 1);
      mbar_init(&pf[2 * i], 8);  // the first and the second 32 keys of both warps of a row
      mbar_init(&pf[2 * i + 1], 8);
      mbar_init(&fin[i], 1);
      mbar_init(&nf[i], 1);
      mbar_init(&ne[i], 17);
    }
    limits[0] = 0;
    limits[1] = 0xffffffffu;
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w.k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w.v) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&w.qm) : "memory");
  }
  if (threadIdx.x >= 64 && threadIdx.x < 64 + PT_ROWS) {
    const uint32_t row = threadIdx.x - 64;
    sts(sm + ROWS + row * 4, row / group | row % group << 16);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, PT_TMEM);
    tmem_relinquish();
  }
  pdl_launch_dependents();
  pdl_wait();
  // ---- what there is to do: every sequence's rows, the places of its blocks, their largest and smallest
  const uint32_t max_len = w.c.ld_table * w.c.page;
  for (uint32_t b = threadIdx.x; b < w.r.batch; b += PT_THREADS) seqs[b] = paged_seq(w.r, max_len, b);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  for (uint32_t b = warp; b < w.r.batch; b += PT_THREADS / 32) {
    const PagedSeq s = seqs[b];
    const uint32_t blocks = (s.rows + 2 * TT - 1) / (2 * TT);
    uint32_t sum = 0, most = 0, least = 0xffffffffu;
    for (uint32_t j = lane; j < blocks; j += 32) {
      const uint32_t n = places_of(block_of(s, j, TT, w.window));
      sum += n;
      most = max(most, n);
      least = min(least, n);
    }
    const uint32_t all = __reduce_add_sync(0xffffffffu, sum);
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) {
      prefix[b + 1] = all * G;
      blocks_in[b] = blocks;
      atomicMax(&limits[0], most);
      atomicMin(&limits[1], least);
    }
  }
  __syncthreads();
  if (warp == 0) {
    uint32_t places = 0, blocks = 0;
    for (uint32_t b = lane; b < w.r.batch; b += 32) {
      places += prefix[b + 1];
      blocks += blocks_in[b];
    }
    places = __reduce_add_sync(0xffffffffu, places);
    blocks = __reduce_add_sync(0xffffffffu, blocks) * G;
    // Whole blocks, taken one by one, end when the last one taken does; equal shares of all places end together, but their blocks have to be joined.
    // Prompt of 2048, 32 heads: 45 us by blocks, 60 by shares; eight drafts of five tokens: 25 and 20.5; three portions and 21 single tokens: 248 and 235.
    const uint32_t ends = blocks <= N ? limits[0] : max(limits[0], places / N + limits[1]);
    const bool shares = ends > places / N + PT_JOIN;
    uint32_t sum = 0;
    for (uint32_t b0 = 0; b0 < w.r.batch; b0 += 32) {
      uint32_t v = 0;
      if (b0 + lane < w.r.batch) v = shares ? prefix[b0 + lane + 1] : blocks_in[b0 + lane] * G;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      if (b0 + lane < w.r.batch) prefix[b0 + lane + 1] = sum + v;
      sum += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) {
      prefix[0] = 0;
      limits[0] = shares;
    }
  }
  __syncthreads();
  const bool shares = limits[0] != 0;
  const uint32_t total = prefix[w.r.batch], share = shares ? max((total + N - 1) / N, PT_LIST1 + 2 * PT_TILE1) : 0;
  // The next segment, in shared memory until `done`.  Warps that meet in barriers go on or end together (`together`), whatever became of a wait.
  uint32_t had = 0;
  auto next = [&](bool &ok, auto together) -> uint32_t {  // its address, 0: there is none
    const uint32_t x = had & 1, at = sm + SEGMENTS + x * (uint32_t)sizeof(Segment);
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(sm + (NF + x) * 8, had >> 1 & 1, sm + ABORT, 980 + x));
    ok = together(ok);
    return ok && lds(at + offsetof(Segment, more)) ? at : 0;
  };
  auto done = [&] {
    __syncwarp();
    if (lane == 0) arrive(sm + (NE + (had & 1)) * 8);
    ++had;
  };

  const bool leader = elect_one();
  if (warp == 0) {
    Finder find(w, prefix, seqs, share);
    const uint32_t box = min(w.c.page, PT_KEYS), boxes = PT_KEYS / box;
    uint32_t it = 0, loads0 = 0, loads1 = 0, handed = 0;
    bool ok = true;
    // Blocks are taken from a counter in the workspace as the copies of the one before end; the CTA that draws the last number sets it back.
    auto take = [&]() -> const Segment * {
      const uint32_t x = handed & 1;
      Segment g;
      bool more;
      if (shares) {
        more = find.part(g);
      } else {
        uint32_t id = blockIdx.x;
        if (handed) {
          if (lane == 0) {
            id = atomicAdd(w.tickets + PAGED_COUNTER, 1u);
            if (id + 1 == total) w.tickets[PAGED_COUNTER] = 0;
            id += N;
          }
          id = __shfl_sync(0xffffffffu, id, 0);
        }
        more = id < total;
        if (more) find.block(id, g);
      }
      if (ok) ok = mbar_wait(sm + (NE + x) * 8, (handed >> 1 & 1) ^ 1, sm + ABORT, 985);
      __syncwarp();
      ++handed;
      if (lane == 0) {
        segments[x] = g;
        segments[x].more = more;
        mbar_arrive(&nf[x]);
      }
      __syncwarp();
      return more ? segments + x : nullptr;
    };
    auto page_of = [&](const Segment *g, uint32_t t, uint32_t end) {
      const uint32_t p = t * PT_KEYS + lane * box;
      return lane < boxes && t < end && p < g->s.len ? __ldcg(w.c.table + (size_t)g->b * w.c.ld_table + p / w.c.page) : -1;
    };
    // Queries of the two halves take the place of the block before's, each when its last scores have been made; the copies of keys and values do not wait for that.
    const Segment *asking = nullptr;
    uint32_t asked = 0;  // bits: halves whose queries have been asked for
    auto ask = [&](uint32_t i, uint32_t &loads) {
      if (asking->k.tokens[i] == 0) {
        asked |= 1u << i;
      } else if (!(asked >> i & 1) && __any_sync(0xffffffffu, test(sm + (QE + i) * 8, (loads & 1) ^ 1))) {
        asked |= 1u << i;
        ++loads;
        if (leader && ok) {
          mbar_arrive_expect_tx(&qf[i], SD * 128 * group * TT);
          for (uint32_t c = 0; c < SD; ++c)
            tma_load_3d(qs + i * UNIT + c * PT_SLAB, &w.qm, (int)(c * 64), (int)(asking->g * group), (int)(asking->s.first + asking->k.token0 + i * TT), &qf[i]);
        }
        __syncwarp();
      }
    };
    auto ask_both = [&] {
      if (asked != 3) {
        ask(0, loads0);
        ask(1, loads1);
      }
    };
    // Until the barrier's phase is over (bar 0: until both halves' queries have been asked for).
    auto wait_asking = [&](uint32_t bar, uint32_t parity, int code) {
      const long long since = clock64();
      bool over = false;
      while (ok && !over) {
        ask_both();
        over = bar ? __all_sync(0xffffffffu, asked == 3 ? try_wait(bar, parity) : test(bar, parity)) : asked == 3;
        if (!over && clock64() - since > WAIT_LIMIT_CYCLES) sts(sm + ABORT, code);
        __syncwarp();
        if (!over && lds(sm + ABORT)) ok = false;
        ok = __all_sync(0xffffffffu, ok);
      }
    };
    const Segment *g = take();
    bool first = true;
    while (g) {
      const uint32_t t0 = g->k.t0, t1 = g->k.t1;
      int ahead = page_of(g, t0, t1);
      asking = g;
      asked = 0;
      if (first) ask_both();
      for (uint32_t t = t0; t < t1; ++t) {
        const int id = ahead;
        ahead = page_of(g, t + 1, t1);
        const uint32_t p = t * PT_KEYS + lane * box;
        // no page: rows in front of the pool, which read as zeros
        const int row = (uint32_t)id < w.c.pages ? (int)(((uint32_t)id * G + g->g) * w.c.page + p % w.c.page) : -(int)PT_KEYS;
#pragma unroll
        for (uint32_t kv = 0; kv < 2; ++kv, ++it) {
          const uint32_t st = it % PT_UNITS;
          wait_asking(sm + (EMPTY + st) * 8, ((it / PT_UNITS) & 1) ^ 1, 900 + st);
          __syncwarp();
          if (leader && ok) mbar_arrive_expect_tx(&full[st], UNIT);
          __syncwarp();
          if (ok && lane < boxes)
            for (uint32_t c = 0; c < SD; ++c) tma_load_2d(ring + st * UNIT + c * PT_SLAB + lane * box * 128, kv ? &w.v : &w.k, (int)(c * 64), row, &full[st]);
        }
      }
      wait_asking(0, 0, 990);
      first = false;
      g = take();
    }
    if (leader && *abort_flag) drain_copies(full, it, PT_UNITS);
    if (leader && *abort_flag) drain_copies(qf, loads0, 1);
    if (leader && *abort_flag) drain_copies(qf + 1, loads1, 1);
  } else if (warp == 1) {
    constexpr uint32_t idesc_s = BF16 ? instr_desc_bf16(PT_ROWS, PT_KEYS) : instr_desc_f16(PT_ROWS, PT_KEYS);
    constexpr uint32_t idesc_o = (BF16 ? instr_desc_bf16(PT_ROWS, DH) : instr_desc_f16(PT_ROWS, DH)) | (1u << 16);  // values: keys are the rows of memory (N-major operand)
    const uint32_t q_lo = smem_desc_lo(smem_u32(qs)), k_lo = smem_desc_lo(smem_u32(ring));
    const uint32_t v_lo = ((smem_u32(ring) >> 4) & 0x3FFFu) | ((PT_SLAB >> 4) << 16);  // 64-element groups are a slab apart
    bool ok = true;
    uint32_t base = 0;  // units before this segment
    // A half: its tiles in this segment, products with the values made in it, phases of its barriers.  Two of them by name and the code for each: an array that is
    // indexed lies in local memory, whose loads stood between the products.
    struct Half {
      uint32_t lo, hi, made, tiles, loads;
    } first{}, second{};
    while (next(ok, [](bool x) { return x; })) {
      const uint32_t at = sm + SEGMENTS + (had & 1) * (uint32_t)sizeof(Segment);
      const uint32_t t0 = lds(at + offsetof(Segment, k.t0)), t1 = lds(at + offsetof(Segment, k.t1));
      const uint32_t tail = lds(at + offsetof(Segment, tail));
      first.lo = lds(at + offsetof(Segment, k.lo)), first.hi = lds(at + offsetof(Segment, k.hi)), first.made = 0;
      second.lo = lds(at + offsetof(Segment, k.lo) + 4), second.hi = lds(at + offsetof(Segment, k.hi) + 4), second.made = 0;
      for (uint32_t t = t0; t <= t1; ++t) {
        // outputs of tile t - 1, scores of tile t, half by half
        const uint32_t ik = base + 2 * (t - t0), iv = ik - 1, sk = ik % PT_UNITS, sv = iv % PT_UNITS;
        const bool kt = t < t1, vt = t > t0;
        bool have_k = false, have_v = false;
        auto products = [&](auto I, Half &h) {
          constexpr uint32_t i = I.value;
          if (vt && t - 1 >= h.lo && t - 1 < h.hi) {
            if (!have_v) {
              if (ok) ok = mbar_wait(sm + (FULL + sv) * 8, (iv / PT_UNITS) & 1, sm + ABORT, 920);
              __syncwarp();
              have_v = true;
              if (tail && t == t1) {  // what the last page holds behind the sequence's end: zeros
                const uint32_t pieces = tail * 8, from = smem_u32(ring) + sv * UNIT + (PT_KEYS - tail) * 128;
                for (uint32_t x = lane; x < pieces * SD; x += 32) {
                  asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(from + x / pieces * PT_SLAB + x % pieces * 16), "r"(0) : "memory");
                }
                fence_proxy_async();
              }
            }
#pragma unroll
            for (uint32_t part = 0; part < 2; ++part) {
              if (ok) ok = mbar_wait(sm + (PF + 2 * i + part) * 8, h.tiles & 1, sm + ABORT, 930 + 2 * i + part);
              __syncwarp();
              if (leader && ok) {
                tc_fence_after();
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) {
                  const uint32_t k16 = (x >> 1) * 4 + part * 2 + (x & 1);  // a half's probabilities lie in the last 32 of its own 64 columns of scores
                  umma_f16_ts(tmem + 256 + i * 128, tmem + i * 128 + (x >> 1) * 64 + 32 + (part * 2 + (x & 1)) * 8, v_lo + sv * (UNIT / 16) + k16 * (2048 >> 4),
                              SMEM_DESC_HI_SW128, idesc_o, (h.made | part | x) ? 1u : 0u);
                }
              }
            }
            if (leader && ok) {
              if (t == h.hi) umma_commit(&fin[i]);
            }
            ++h.tiles;
            ++h.made;
          }
          if (kt && t >= h.lo && t < h.hi) {
            if (!have_k) {
              if (ok) ok = mbar_wait(sm + (FULL + sk) * 8, (ik / PT_UNITS) & 1, sm + ABORT, 940);
              __syncwarp();
              have_k = true;
            }
            if (t == h.lo) {
              if (ok) ok = mbar_wait(sm + (QF + i) * 8, h.loads & 1, sm + ABORT, 910 + i);
              __syncwarp();
            }
            __syncwarp();
            if (leader && ok) {
              tc_fence_after();
#pragma unroll
              for (uint32_t k16 = 0; k16 < DH / 16; ++k16) {
                umma_f16(tmem + i * 128, q_lo + (i * UNIT + (k16 / 4) * PT_SLAB) / 16 + (k16 & 3) * 2, k_lo + (sk * UNIT + (k16 / 4) * PT_SLAB) / 16 + (k16 & 3) * 2,
                         SMEM_DESC_HI_SW128, idesc_s, k16 ? 1u : 0u);
              }
              umma_commit(&sf[i]);
              if (t + 1 == h.hi) umma_commit(&qe[i]);
            }
          }
        };
        products(std::integral_constant<uint32_t, 0>(), first);
        products(std::integral_constant<uint32_t, 1>(), second);
        // every tile has a half that uses it, so both units have been waited for
        if (leader && ok && vt) umma_commit(&empty[sv]);
        if (leader && ok && kt) umma_commit(&empty[sk]);
      }
      base += 2 * (t1 - t0);
      auto queries_read = [&](auto I, Half &h) {
        constexpr uint32_t i = I.value;
        if (lds(at + offsetof(Segment, k.tokens) + 4 * i)) {
          // Queries of a half without tiles are waited for all the same: no copy outlives the CTA.
          if (h.lo == h.hi) {
            if (ok) ok = mbar_wait(sm + (QF + i) * 8, h.loads & 1, sm + ABORT, 912 + i);
            __syncwarp();
            if (lane == 0) arrive(sm + (QE + i) * 8);
          }
          ++h.loads;
        }
      };
      queries_read(std::integral_constant<uint32_t, 0>(), first);
      queries_read(std::integral_constant<uint32_t, 1>(), second);
      done();
    }
  } else {
    const uint32_t i = (uint32_t)(warp - 2) >> 3, half = ((uint32_t)(warp - 2) >> 2) & 1, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t sb = tmem + (quad * 32 << 16) + i * 128 + half * 64, ob = sb + 256 - half * (64 - DH / 2);  // the thread's scores, and outputs
    const uint32_t mine = sm + MEET + ((i * 2 + half) * PT_ROWS + row) * 4, theirs = mine ^ (PT_ROWS * 4);
    auto meet_other = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + i * 4 + quad) : "memory"); };  // with the other warp of these rows
    auto agree = [&](bool x) {  // whether any thread of the two warps says so
      uint32_t any;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"(1 + i * 4 + quad), "r"((uint32_t)x) : "memory");
      return any != 0;
    };
    auto meet_all = [] { asm volatile("bar.sync 9, 512;" ::: "memory"); };  // all rows' warps
    bool ok = true;
    uint32_t phases = 0;  // of the half's barriers: 1 scores, 2 ends
    // Pairs of warps meet in every tile, all of them where blocks are joined.
    auto together = [&](bool x) {
      if (!lds(sm + WORDS + 8)) return !agree(!x);  // no shares
      uint32_t all;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 9, 512, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"((uint32_t)x) : "memory");
      return all != 0;
    };
    while (const uint32_t g32 = next(ok, together)) {
      const uint32_t of_half = g32 + i * 4;
      const uint32_t tokens = lds(of_half + offsetof(Segment, k.tokens)), lo = lds(of_half + offsetof(Segment, k.lo)), n = lds(of_half + offsetof(Segment, k.hi)) - lo;
      const bool any_live = quad * 32 < tokens * group;
      float m2 = PT_LOWEST, l = 0.f;  // the row's maximum times scale2, less PT_BELOW; the sum of this thread's half
      // What a tile needs of the segment is read from shared memory where it is needed: the row's scores leave no registers for it.
      for (uint32_t t = lo; t < lo + n; ++t) {  // to the end, whatever became of a wait: the two warps of a row meet in every tile
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(sm + (SF + i) * 8, phases & 1, sm + ABORT, 960 + i));
        phases ^= 1;
        tc_fence_after();
        if (!any_live) {  // rows behind the last: their probabilities may be anything
          if (lane == 0) {
            arrive(sm + (PF + 2 * i) * 8);
            arrive(sm + (PF + 2 * i + 1) * 8);
          }
          continue;
        }
        const bool masks = t < lds(of_half + offsetof(Segment, clear0)) || t >= lds(of_half + offsetof(Segment, clear1));
        auto hide = [&](uint32_t (&v)[32], int c) {  // scores of keys that the row does not see
          if (masks) {
            const int pos = row < tokens * group ? (int)lds(of_half + offsetof(Segment, pos)) + (int)(lds(sm + ROWS + row * 4) & 0xffff) : -1, a = (int)(t * PT_KEYS + half * 64 + c * 32);
            const int n0 = w.window ? min(max(pos - (int)w.window + 1 - a, 0), 32) : 0, n1 = min(max(pos + 1 - a, 0), 32);
            const uint32_t seen = (uint32_t)((1ull << n1) - 1) & ~(uint32_t)((1ull << n0) - 1);
            if (!__all_sync(0xffffffffu, seen == 0xffffffffu)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!(seen >> j & 1)) v[j] = 0xFF800000u;
            }
          }
        };
        auto largest = [&](const uint32_t (&v)[32]) {
          float tm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 32; j += 2) tm[(j / 2) & 3] = fmaxf(fmaxf(tm[(j / 2) & 3], __uint_as_float(v[j])), __uint_as_float(v[j + 1]));
          return fmaxf(fmaxf(tm[0], tm[1]), fmaxf(tm[2], tm[3]));
        };
        // Probabilities of 32 scores into 16 columns of tensor memory, 16 scores at a time; their sum.
        auto probabilities = [&](const uint32_t (&v)[32], uint32_t to) {
          uint64_t two[2] = {0, 0};
          const uint64_t scale = pair(w.scale2, w.scale2), minus = pair(-m2, -m2);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 x = unpair(fma2(pair(__uint_as_float(v[h * 16 + 2 * j]), __uint_as_float(v[h * 16 + 2 * j + 1])), scale, minus));
              const float a = ex2(x.x), b = ex2(x.y);
              two[j & 1] = add2(two[j & 1], pair(a, b));
              p[j] = pack2<BF16>(a, b);
            }
            tmem_st8(to + h * 8, p);
          }
          const float2 s0 = unpair(two[0]), s1 = unpair(two[1]);
          return (s0.x + s0.y) + (s1.x + s1.y);
        };
        auto release = [&](int c) {  // the products of the first 32 keys begin while the others' probabilities are made
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive(sm + (PF + 2 * i + c) * 8);
        };
        // The first 32 probabilities are made against the maximum so far; where it has grown too much (a row's two threads have to agree, and the barrier tells
        // both) they are made again, from the scores that still stand: probabilities lie in the columns of the other 32, which are in registers by then.
        const bool start = t == lo;
        uint32_t v[32], u[32];
        tmem_ld32(sb, v);
        tmem_ld32(sb + 32, u);
        tmem_ld_wait();
        hide(v, 0);
        hide(u, 1);
        const float tmax = fmaxf(largest(v), largest(u));
        float sum = 0.f;
        if (!start) sum = probabilities(v, sb + 32);
        if (agree(start || tmax * w.scale2 > m2 + (PT_LAZY + PT_BELOW<BF16>))) {
          sts(mine, __float_as_uint(tmax));
          meet_other();
          const float nm = fmaxf(m2, fmaxf(tmax, __uint_as_float(lds(theirs))) * w.scale2 - PT_BELOW<BF16>);
          const bool grown = start || nm > m2 + PT_LAZY;
          const float f = grown ? ex2(m2 - nm) : 1.f;
          if (grown) m2 = nm;
          l *= f;
          if (!start) {
#pragma unroll 1
            for (uint32_t c = 0; c < DH / 2; c += 8) {
              uint32_t o[8];
              tmem_ld8(ob + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st8(ob + c, o);
            }
          }
          tmem_ld32(sb, v);
          tmem_ld_wait();
          hide(v, 0);
          sum = probabilities(v, sb + 32);
        }
        l += sum;
        release(0);
        l += probabilities(u, sb + 48);
        release(1);
      }
      if (n) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(sm + (FIN + i) * 8, phases >> 1 & 1, sm + ABORT, 970 + i));
        phases ^= 2;
      }
      if (any_live) {
        meet_other();  // the last maximum has been read
        sts(mine, __float_as_uint(l));
        meet_other();
        l += __uint_as_float(lds(theirs));
      }
      tc_fence_after();
      const Segment *g = segments + (had & 1);
      const uint32_t c0 = g->c0, c1 = g->c1;
      const bool whole = g->whole;
      // 32 elements of the thread's row from c on, as they are stored.  16 bytes a lane straight from a row per lane would be a line each: four lanes change places
      // (a 4 x 4 transposition of 16-byte pieces), and store 64 bytes of each of their rows in turn.
      uint16_t *base = static_cast<uint16_t *>(w.o) + (size_t)(g->s.first + g->k.token0 + i * TT) * w.ld_o + (size_t)g->g * group * w.c.dim;
      auto put = [&](const float (&y)[32], uint32_t c, float inv) {
        __syncwarp();
        uint32_t q[4][4];
#pragma unroll
        for (int j = 0; j < 16; ++j) q[j / 4][j & 3] = pack2<BF16>(y[2 * j] * inv, y[2 * j + 1] * inv);
#pragma unroll
        for (int s = 1; s < 4; s *= 2)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (!(x & s)) {
              const bool up = lane & s;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? q[x][j] : q[x + s][j], s);
                if (up)
                  q[x][j] = got;
                else
                  q[x + s][j] = got;
              }
            }
        const uint32_t e = c + (lane & 3) * 8;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t r = (row & ~3u) + x;
          if (r >= tokens * group || e >= w.c.dim || !ok) continue;
          const uint32_t at = lds(sm + ROWS + r * 4);
          *reinterpret_cast<uint4 *>(base + (size_t)(at & 0xffff) * w.ld_o + (at >> 16) * w.c.dim + e) = make_uint4(q[x][0], q[x][1], q[x][2], q[x][3]);
        }
      };
      // A part: [maxima][sums][4 elements][row], rows of both halves.
      auto part_of = [&](uint32_t cta) { return w.parts + (size_t)(2 * cta + (cta == c0 ? 1 : 0)) * PAGED_PART; };
      const uint32_t r2 = i * PT_ROWS + row;
      float *own = whole ? nullptr : part_of(blockIdx.x);
      float inv = m2 == PT_LOWEST ? 0.f : 1.f / l;  // a row that has seen no score: zeros
      if (any_live) {
#pragma unroll 1
        for (uint32_t c = half * (DH / 2); c < (half + 1) * (DH / 2); c += 32) {
          float y[32], z = 0.f;  // z: 0, or NaN
          if (n) {
            uint32_t o[32];
            __syncwarp();
            tmem_ld32(ob + c - half * (DH / 2), o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              y[j] = __uint_as_float(o[j]);
              z = fmaf(y[j], 0.f, z);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j] = 0.f;
          }
          if (z != 0.f && row < tokens * group && isfinite(l)) {
            const int pos = g->pos[i] + (int)(row / group);
            float x[32];  // in memory, which `y` stays out of
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = y[j];
            paged_again<32>(w, BF16, false, g->b, g->s, g->g, (g->k.token0 + i * TT) * group + row, [&](int j) { return c + j; }, max(w.window ? pos - (int)w.window + 1 : 0, (int)(lo * PT_KEYS)),
                            min(pos + 1, (int)min((lo + n) * PT_KEYS, 0x7fffffffu)), m2, 1.f, x);
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j] = x[j];
          }
          if (whole) {
            put(y, c, inv);
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              __stcg(reinterpret_cast<float4 *>(own + 4 * PT_ROWS) + (c + j) / 4 * (2 * PT_ROWS) + r2, make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]));
          }
        }
      }
      if (!whole) {
        if (half == 0) {
          __stcg(own + r2, m2);
          __stcg(own + 2 * PT_ROWS + r2, l);
        }
        __threadfence();
        meet_all();
        if (warp == 2 && lane == 0) {
          const uint32_t before = atomicAdd(w.tickets + c0, 1u);
          if (before == c1 - c0) w.tickets[c0] = 0;  // all are here: the ticket is free again
          *ticket = before;
          __threadfence();
        }
        meet_all();
        if (lds(sm + WORDS + 4) == c1 - c0 && any_live) {  // the last: joins the parts in the order of their tiles
          float big = PT_LOWEST;
          for (uint32_t x = c0; x <= c1; ++x) big = fmaxf(big, __ldcg(part_of(x) + r2));
          l = 0.f;
          for (uint32_t x = c0; x <= c1; ++x) l = fmaf(__ldcg(part_of(x) + 2 * PT_ROWS + r2), ex2(__ldcg(part_of(x) + r2) - big), l);
          inv = big == PT_LOWEST ? 0.f : 1.f / l;
#pragma unroll 1
          for (uint32_t c = half * (DH / 2); c < (half + 1) * (DH / 2); c += 32) {
            float y[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j] = 0.f;
#pragma unroll 1
            for (uint32_t x = c0; x <= c1; ++x) {
              const float *from = part_of(x);
              const float f = ex2(__ldcg(from + r2) - big);
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 o = __ldcg(reinterpret_cast<const float4 *>(from + 4 * PT_ROWS) + (c + j) / 4 * (2 * PT_ROWS) + r2);
                y[j] = fmaf(o.x, f, y[j]);
                y[j + 1] = fmaf(o.y, f, y[j + 1]);
                y[j + 2] = fmaf(o.z, f, y[j + 2]);
                y[j + 3] = fmaf(o.w, f, y[j + 3]);
              }
            }
            put(y, c, inv);
          }
        }
      }
      tc_fence_before();  // the outputs have been read: the next products may take their place
      done();
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
int launch_tc(cudaStream_t stream, const PagedAttnArgs &w) {
  const size_t fixed = (size_t)(2 + PT_UNITS) * SD * PT_SLAB + 1024 + PT_SMALL + 8, per = 8 + sizeof(PagedSeq);
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    GRETA_CUDA_TRY(cudaFuncSetAttribute(paged_tc_kernel<SD, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(fixed + PAGED_MAX_BATCH * per)));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const uint32_t grid = std::min<uint32_t>(PT_MAX_CTAS, sm_count());  // one a SM: its tensor memory and most of its shared memory
  GRETA_CUDA_TRY(launch_pdl(paged_tc_kernel<SD, BF16>, dim3(grid), dim3(PT_THREADS), fixed + w.r.batch * per, stream, w));
  return launched("paged_tc_kernel");
}

}  // namespace

namespace greta {

// Places are numbered with 32 bits, of whatever lengths the tables have room for: about a second's work.
bool paged_tc_fits(const PagedAttnArgs &w) {
  if (w.group > PT_ROWS) return false;
  const uint64_t blocks = w.r.tokens / (2 * (PT_ROWS / w.group)) + std::min(w.r.batch, w.r.tokens), tiles = (uint64_t)w.c.ld_table * w.c.page / PT_KEYS + 1;
  return blocks * w.c.kv_heads < (1ull << 31) / (tiles * PT_TILE2 + PT_LIST2);
}
// Queries of the cache's type, where paged_tc_fits; w.k and w.v with boxes of min(page, 128) rows.
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
  if (d > 64) return bf16 ? launch_tc<2, true>(stream, w) : launch_tc<2, false>(stream, w);
  return bf16 ? launch_tc<1, true>(stream, w) : launch_tc<1, false>(stream, w);
}

}  // namespace greta
