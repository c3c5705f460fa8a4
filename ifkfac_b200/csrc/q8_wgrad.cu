// Weight and bias gradient of a linear layer from its 8-bit input rows
// (ifk_q8_wgrad): dW = delta^T X, db = column sums of delta.
//
// dW is a matrix product whose long axis is the rows, so both operands are
// M/N-major: a row of delta or of X is contiguous along the output.  The 8-bit
// rows take the M side (128 input columns a CTA), delta the N side (256 output
// columns), so the accumulator in TMEM has an input column a lane and the
// epilogue's stores are contiguous along dW's rows.
//
// A pair of CTAs shares one 256 x 256 tile (tcgen05 cta_group::2).  Per step of 64
// rows each CTA brings half of delta's columns (bf16) and its own 128 columns of codes
// by TMA, four warps turn the codes into a bf16 tile, and one thread of the pair issues
// the step's four tcgen05.mma.  A code times its power-of-two scale is exact in bf16,
// so the products are exact and only the fp32 sums round.  An fp32 delta is taken apart
// beforehand into three bf16 terms (8 + 8 + 8 bits, by truncation: exact), and each 64
// rows take three steps.
//
// The tensor core truncates as it adds to the accumulator, so a long sum drifts towards
// zero: positive codes and deltas over 16384 rows come out 6.1e-5 low, over 65536 rows
// 3.5e-4 (random signs, 16384 rows: 7e-6).  After CHUNK steps (120 tcgen05.mma) the
// accumulator is therefore added to dW in L2 (red.global.add, rounded to nearest; one
// thread owns an element, so the order is fixed) while the next chunk goes to the other
// half of TMEM: 1.1e-6 low in bf16 at either length, 1.5e-6 at most; in the three terms
// of an fp32 delta 4e-8, 7e-7 at most.
//
// Work: whole waves of tiles first, every cluster a tile at a time; the tiles that
// are left over are cut along the rows into equal shares for all clusters.  A share
// that is not a whole tile goes to the workspace, and a second kernel adds a
// tile's shares in order.
//
// Bound by shared memory's port: a step moves 98 KB through it in each SM (codes in and
// out, the tile out and into the tensor core, delta's half in and twice out), 765 clocks
// where the tensor core needs 512.  Measured: 16384 x 4096 x 4096 bf16 435 to 470 us (1.2
// PFLOP/s at the 1.5 GHz that the card's power allows) and 36 us for db's sums and the
// join, 470 to 485 us in all where a graph's calls follow one another and 545 to 572 us
// with every call's inputs from memory; 8192 x 768 x 2304 34 + 16 us (49 in all); one row of 2048 x 8192 17 us (67 MB written);
// 8192 x 4096 x 4096 fp32 720 to 750 us in all.  A launch's fixed part is about 6 us: set-up 1, the
// first loads 2, the last accumulator's stores 2, the pair's last meeting 1.
#include <cuda.h>

#include <algorithm>
#include <cstring>

#include "rowvec.cuh"
#include "ifk_internal.h"
#include "pipe.cuh"
#include "tc.cuh"

namespace ifk {

namespace {

constexpr int KS = 64;        // rows a step
constexpr int TM = 128;       // input columns a CTA
constexpr int TN = 256;       // output columns a tile
constexpr int CHUNK = 30;     // steps a TMEM accumulator sums: 30 row blocks, or 10 in three terms
constexpr int CONV_WARPS = 4;   // converting warps of a step
constexpr int CONV_GROUPS = 4;  // such groups, taking turns
// warps: 0 delta, 1 MMA, 2 TMEM and codes, 3 scales, 4-7 epilogue, 8 .. conversion
constexpr int THREADS = 32 * (8 + CONV_WARPS * CONV_GROUPS);
constexpr int SM_COUNT = 148, CLUSTERS = SM_COUNT / 2;
constexpr int MIN_STEPS = 4;  // least steps a share of a cut tile is worth
constexpr uint32_t ATOM = 64 * KS * 2;  // 64 columns (128 bytes) of KS rows

// Shared memory: a ring of NS steps (a converted tile and delta's half each), a ring of
// NC steps of codes and scales, the barriers.  A load takes about a microsecond, a step at
// the tensor core's rate a third of one.
constexpr int NS = 6, NC = 4;
// A parity wait also passes one phase early, so whoever waits on a barrier has to have seen
// the phase before.  A converting group's slots of codes are its own; and before it writes
// a tile, step i waits for the products of step i - NS, of which the phase before is step
// i - 2 NS, while the group's last step has waited for step i - NS - CONV_GROUPS.
static_assert(NC == CONV_GROUPS && CONV_GROUPS <= NS, "rings and groups");
constexpr uint32_t A_BYTES = TM * KS * 2, D_BYTES = TN / 2 * KS * 2, C_BYTES = TM * KS;
constexpr uint32_t O_TILES = 0, O_DELTA = O_TILES + NS * A_BYTES, O_CODES = O_DELTA + NS * D_BYTES;
constexpr uint32_t O_SCALES = O_CODES + NC * C_BYTES;  // per slot KS x 4 bytes
constexpr uint32_t O_BARS = O_SCALES + NC * KS * 4;
constexpr int NBARS = 2 * NC + 2 * NS + 4;
static_assert(NBARS <= 32, "a lane sets up a barrier");
constexpr uint32_t SMEM = O_BARS + NBARS * 8 + 16;

// Division of the tiles between clusters.
struct Plan {
  int Ti, To;          // tiles along the input and output columns
  int Kt;              // steps a tile
  int G;               // clusters
  int Tdp;             // tiles done whole, in waves
  int Gs;              // clusters that share the rest
  int64_t total;       // steps of the rest
  __host__ __device__ int64_t share(int c) const { return total * c / Gs; }
  // the cluster whose share holds step p of the rest
  __host__ __device__ int owner(int64_t p) const { return (int)(((p + 1) * Gs - 1) / total); }
};

struct Args {
  Plan p;
  int terms;           // bf16 terms of delta
  const uint8_t* scales;
  int64_t lds, rows, n_out, n_in, ldw;
  float* dW;
  float* part;         // [2 Gs][TN][2 TM]
  int accumulate;
  bool vec_scales;     // rows of scales start at multiples of 4 bytes
  bool vec_out;        // rows of dW start at multiples of 16 bytes
  bool copied;         // delta's terms are written by the pass before
  bool whole;          // delta's map has 64-column blocks as a dimension (n_out a multiple of 64)
  int* status;
  bool withhold;       // tests only (IFK_DEBUG_WITHHOLD): the second CTA's first codes never count as landed
};

// The steps of a tile in order: which block of KS rows, and which of delta's terms.  The terms of
// a chunk's rows come smallest first, so that the sums of the small ones are truncated
// at their own size.  Kept from step to step, as one thread issues the copies: with the divisions
// of a step's place each time, 8192 x 4096 x 4096 fp32 took 850 us instead of 750.
struct Steps {
  int base, nb, i, q, blocks, terms;  // a chunk's first block and their number, the block in it, the pass over them
  __device__ __forceinline__ Steps(const Args& a, int k) : base(k), nb(0), i(0), q(0), blocks(0), terms(a.terms) {
    if (terms == 1) return;
    blocks = a.p.Kt / 3;
    const int sup = k / CHUNK, rem = k - sup * CHUNK;
    base = sup * (CHUNK / 3);
    nb = mn(CHUNK / 3, blocks - base);
    q = rem / nb;
    i = rem - q * nb;
  }
  __device__ __forceinline__ int block() const { return base + i; }
  __device__ __forceinline__ int term() const { return terms == 1 ? 0 : 2 - q; }
  __device__ __forceinline__ void next() {
    ++i;
    if (terms == 1 || i < nb) return;
    i = 0;
    if (++q < 3) return;
    q = 0;
    base += CHUNK / 3;
    nb = mn(CHUNK / 3, blocks - base);
  }
};
// End of the chunk that step k is in.
__device__ __forceinline__ int chunk_end(int k, int k1) { return mn((k / CHUNK + 1) * CHUNK, k1); }

// One piece of work: steps k0 .. k1 of a tile; slot < 0: the whole tile.
struct Piece {
  int tile, k0, k1, slot;
};

// Position in a ring of N slots: the slot and the parity of its round.
template <int N>
struct Ring {
  uint32_t s = 0, ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      ph ^= 1;
    }
  }
};

// The pieces of cluster c in order.
struct Walk {
  const Plan& p;
  int c, next_tile;
  int64_t at, end;
  __device__ Walk(const Plan& plan, int cluster) : p(plan), c(cluster), next_tile(cluster), at(0), end(0) {
    if (c < p.Gs && p.total > 0) {
      at = p.share(c);
      end = p.share(c + 1);
    }
  }
  __device__ int64_t steps() const {
    return (c < p.Tdp ? (int64_t)((p.Tdp - 1 - c) / p.G + 1) * p.Kt : 0) + (end - at);
  }
  __device__ bool next(Piece& w) {
    if (next_tile < p.Tdp) {
      w.tile = next_tile;
      w.k0 = 0;
      w.k1 = p.Kt;
      w.slot = -1;
      next_tile += p.G;
      return true;
    }
    if (at >= end) return false;
    const int64_t t = at / p.Kt, b = t * p.Kt;
    w.tile = p.Tdp + (int)t;
    w.k0 = (int)(at - b);
    w.k1 = (int)(mn<int64_t>(b + p.Kt, end) - b);
    // a piece that starts inside its tile is the first of its cluster, one that only ends inside it the last
    w.slot = w.k0 > 0 ? 2 * c : (w.k1 < p.Kt ? 2 * c + 1 : -1);
    at = b + w.k1;
    return true;
  }
};

// ---- PTX ----

// The address of the same place in the pair's first CTA.
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// A copy into this CTA's memory that completes on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_4d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int t,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(t), "r"(bar)
      : "memory");
}

// The kernels of a call follow one another; one that is launched behind the last (programmatic stream
// serialisation) may start and set itself up once every block of the last has run let_next_start or has ended, and
// wait_for_last holds it until the last is done and its writes are visible.  Each waits before it ends, so the
// end of a call's last kernel is the end of all of them; the first is launched as usual, after all before it.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void red_add(float* p, float v) {
  asm volatile("red.global.add.f32 [%0], %1;" ::"l"(p), "f"(v) : "memory");
}

// Operand tiles: M/N-major, 128-byte swizzle.  64 columns of 8 rows are one 1024-byte
// atom; the next 8 rows follow at SBO = 1024 bytes, the next 64 columns at LBO = ATOM.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(ATOM >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// D (+)= A B over the pair's two halves; issued by one thread of its first CTA.
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}

// Arrive on this barrier in both CTAs when the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}

// The pair's barrier in two halves; whole warps, one wait after each arrival.
__device__ __forceinline__ void pair_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void pair_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Four packed codes to four bf16 values, exactly.  With the byte's low seven bits under
// the exponent of 128, 128 + low; 128 + (sign bit) is the other term; their difference is the code.
__device__ __forceinline__ void codes4(uint32_t w, __nv_bfloat162 scale, uint32_t& lo, uint32_t& hi) {
  const uint32_t t[2] = {__byte_perm(w, 0u, 0x4140), __byte_perm(w, 0u, 0x4342)};
  uint32_t r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t a = (t[i] & 0x007f007fu) | 0x43004300u, b = (t[i] & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                             *reinterpret_cast<const __nv_bfloat162*>(&b)), scale);
    r[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  lo = r[0];
  hi = r[1];
}

__global__ void __launch_bounds__(THREADS, 1)
wgrad_kernel(const __grid_constant__ CUtensorMap dmap, const __grid_constant__ CUtensorMap cmap, const Args a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = tc::smem_u32(smem);
  // codes_full: codes and scales have landed; codes_free: they are converted;
  // ready (first CTA): both CTAs' tiles are converted and both halves of delta have landed;
  // free: the step is multiplied; acc_full / acc_free: an accumulator is summed / read
  const uint32_t codes_full = base + O_BARS, codes_free = codes_full + 8 * NC;
  const uint32_t ready = codes_free + 8 * NC, free = ready + 8 * NS, acc_full = free + 8 * NS, acc_free = acc_full + 16;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + O_BARS + NBARS * 8);
  volatile int* failed = reinterpret_cast<volatile int*>(slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x & 1;
  const int cluster = blockIdx.x >> 1;

  // what a role has to compute (divisions) and fetch before its first copy, while the barriers are set up
  if (lane == 0 && warp == 0) prefetch_map(&dmap);
  if (lane == 0 && warp == 2) prefetch_map(&cmap);
  Walk walk(a.p, cluster);
  const int64_t steps = walk.steps();
  Piece w;
  bool more = walk.next(w);

  if (warp == 1) {
    if (lane == 0) *failed = 0;
    // the arrivals that a phase takes; codes_full: the copy, and the lanes that bring the scales; codes_free:
    // a group's warps; ready: the copies, and both CTAs' warps of a group; free and acc_full: the products;
    // acc_free: both CTAs' reading warps
    int i = lane, arrivals = 4 * 2;
    if (i < NC) arrivals = 1 + 32 + (a.withhold && blockIdx.x == 1 && i == 0 ? 1 : 0);
    else if (i < 2 * NC) arrivals = CONV_WARPS;
    else if (i < 2 * NC + NS) arrivals = 1 + CONV_WARPS * 2;
    else if (i < 2 * NC + 2 * NS + 2) arrivals = 1;
    if (i < NBARS) tc::mbar_init(reinterpret_cast<uint64_t*>(smem + O_BARS) + i, arrivals);
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc::smem_u32(slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *slot;
  // the warps that fetch codes and scales need this CTA's barriers alone: they wait for the other's at the end
  pair_arrive();
  if (warp != 2 && warp != 3) pair_wait();

  if (warp == 0) {
    if (lane == 0) {
      Ring<NS> r;
      const uint32_t bar0 = in_leader(ready);
      bool ok = true, now = true;
      if (a.copied) wait_for_last();
      for (; ok && more; more = walk.next(w)) {
        const int o = w.tile / a.p.Ti * TN + (int)rank * (TN / 2);
        Steps sp(a, w.k0);
        for (int k = w.k0; k < w.k1; ++k, sp.next()) {
          if (!now && !wait_bar(free + 8 * r.s, r.ph ^ 1, failed)) {
            ok = false;
            break;
          }
          const uint32_t dst = base + O_DELTA + r.s * D_BYTES, bar = bar0 + 8 * r.s;
          if (rank == 0) expect(ready + 8 * r.s, 2 * D_BYTES);  // both CTAs' copies
          if (a.whole) {
            tma_4d_pair(dst, &dmap, 0, sp.block() * KS, o >> 6, sp.term(), bar);
          } else {
            tma_4d_pair(dst, &dmap, o, sp.block() * KS, 0, sp.term(), bar);
            tma_4d_pair(dst + ATOM, &dmap, o + 64, sp.block() * KS, 0, sp.term(), bar);
          }
          r.next();
          now = test_bar(free + 8 * r.s, r.ph ^ 1);
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc = tc::idesc_bf16(TM * 2, TN, true, true);
      const uint64_t ad0 = desc_sw128(base + O_TILES), bd0 = desc_sw128(base + O_DELTA);
      Ring<NS> r;
      uint32_t buf = 0, bph = 0;
      bool ok = true, now = false;
      for (; ok && more; more = walk.next(w)) {
        for (int c0 = w.k0, c1; ok && c0 < w.k1; c0 = c1) {
          c1 = chunk_end(c0, w.k1);
          if (!wait_bar(acc_free + 8 * buf, bph ^ 1, failed)) {
            ok = false;
            break;
          }
          tc::fence_after();
          const uint32_t acc = tmem + buf * TN;
          for (int k = c0; k < c1; ++k) {
            if (!now && !wait_bar(ready + 8 * r.s, r.ph, failed)) {
              ok = false;
              break;
            }
            tc::fence_after();
            const uint64_t ad = ad0 + tc::doff(r.s * A_BYTES), bd = bd0 + tc::doff(r.s * D_BYTES);
            const uint32_t bar = free + 8 * r.s;
            r.next();
            mma_pair(acc, ad, bd, idesc, k > c0 ? 1u : 0u);
            mma_pair(acc, ad + tc::doff(2048), bd + tc::doff(2048), idesc, 1u);
            now = test_bar(ready + 8 * r.s, r.ph);  // the next step's, while this one's products are issued
            mma_pair(acc, ad + tc::doff(2 * 2048), bd + tc::doff(2 * 2048), idesc, 1u);
            mma_pair(acc, ad + tc::doff(3 * 2048), bd + tc::doff(3 * 2048), idesc, 1u);
            commit_pair(bar);
          }
          if (ok) commit_pair(acc_full + 8 * buf);
          buf ^= 1;
          if (buf == 0) bph ^= 1;
        }
      }
    }
  } else if (warp == 2) {
    if (lane == 0) {
      Ring<NC> r;
      bool ok = true, now = true;
      for (; ok && more; more = walk.next(w)) {
        const int x = (w.tile % a.p.Ti * 2 + (int)rank) * TM;
        Steps sp(a, w.k0);
        for (int k = w.k0; k < w.k1; ++k, sp.next()) {
          if (!now && !wait_bar(codes_free + 8 * r.s, r.ph ^ 1, failed)) {
            ok = false;
            break;
          }
          expect(codes_full + 8 * r.s, C_BYTES);
          tma_2d(base + O_CODES + r.s * C_BYTES, &cmap, x, sp.block() * KS, codes_full + 8 * r.s);
          r.next();
          now = test_bar(codes_free + 8 * r.s, r.ph ^ 1);
        }
      }
    }
  } else if (warp == 3) {
    // the scale bytes of a slot: rows lane and lane + 32, four groups each; a row past the end has zeros
    Ring<NC> r;
    bool ok = true;
    const int64_t groups = q8::pitch(a.n_in) / q8::GROUP;
    for (; ok && more; more = walk.next(w)) {
      const int64_t gi = (int64_t)(w.tile % a.p.Ti * 2 + (int)rank) * (TM / q8::GROUP);
      const bool vec = a.vec_scales && gi + 4 <= groups;
      Steps sp(a, w.k0);
      // this lane's two rows of a step
      auto source = [&](int h) {
        const int64_t row = (int64_t)sp.block() * KS + h * 32 + lane;
        return row < a.rows ? a.scales + row * a.lds + gi : nullptr;
      };
      const uint32_t at = O_SCALES + lane * 4;
      if (vec) {
        for (int k = w.k0; k < w.k1; ++k, r.next(), sp.next()) {
          if (!wait_bar(codes_free + 8 * r.s, r.ph ^ 1, failed)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t* p = source(h);
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(base + at + r.s * (KS * 4) + h * 128),
                         "l"(p ? p : a.scales), "r"(p ? 4 : 0)
                         : "memory");
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(codes_full + 8 * r.s) : "memory");
        }
      } else {
        // byte by byte, two steps ahead: waiting for each step's bytes took 1500 clocks a step
        uint32_t v[2][2][4];
        auto fetch = [&](uint32_t (&q)[2][4]) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t* p = source(h);
#pragma unroll
            for (int g = 0; g < 4; ++g) q[h][g] = p && gi + g < groups ? p[g] : 0u;
          }
          sp.next();
        };
        fetch(v[0]);
        if (w.k0 + 1 < w.k1) fetch(v[1]);
        for (int k = w.k0; ok && k < w.k1; k += 2) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (k + e >= w.k1) break;
            if (!wait_bar(codes_free + 8 * r.s, r.ph ^ 1, failed)) {
              ok = false;
              break;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
              *reinterpret_cast<uint32_t*>(smem + at + r.s * (KS * 4) + h * 128) =
                  v[e][h][0] | v[e][h][1] << 8 | v[e][h][2] << 16 | v[e][h][3] << 24;
            arrive(codes_full + 8 * r.s);
            r.next();
            if (k + e + 2 < w.k1) fetch(v[e]);
          }
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= 4 && warp < 8) {
    uint32_t buf = 0, bph = 0;
    const int wq = warp & 3;  // the quarter of TMEM's lanes this warp reads
    bool ok = true;
    for (; ok && more; more = walk.next(w)) {
      const int ti = w.tile % a.p.Ti, to = w.tile / a.p.Ti;
      const int m = (int)rank * TM + wq * 32 + lane;
      const int64_t i = (int64_t)ti * 2 * TM + m, o0 = (int64_t)to * TN;
      // where this thread's column of the tile goes: dW, or its share's slot
      const bool to_part = w.slot >= 0;
      float* d = to_part ? a.part + (int64_t)w.slot * (TN * 2 * TM) + m : a.dW + o0 * a.ldw + i;
      const int64_t ld = to_part ? 2 * TM : a.ldw;
      const bool in = i < a.n_in;
      // columns of the tile that dW has (none where the whole warp is past its rows' end)
      const int cols = i - lane < a.n_in ? (int)mn<int64_t>(TN, a.n_out - o0) : 0;
      bool add = !to_part && a.accumulate;
      for (int c0 = w.k0; c0 < w.k1; c0 = chunk_end(c0, w.k1)) {
        if (!wait_bar(acc_full + 8 * buf, bph, failed)) {
          if (in) *d = __int_as_float(0x7fffffff);  // a sum that is not whole: NaN in the first row of the piece
          ok = false;
          break;
        }
        tc::fence_after();
        for (int c = 0; c < cols; c += 32) {
          float v[32];
          tc::tmem_ld32(tmem + buf * TN + c + ((uint32_t)(wq * 32) << 16), v);
          float* p = d + c * ld;
          if (!in) continue;
          if (c + 32 <= cols) {
            // four addresses, so that the next one does not wait for the last
            float* at[4] = {p, p + ld, p + 2 * ld, p + 3 * ld};
            const int64_t ld4 = 4 * ld;
            if (add) {
#pragma unroll
              for (int q = 0; q < 32; ++q, at[(q + 3) & 3] += ld4) red_add(at[q & 3], v[q]);
            } else {
#pragma unroll
              for (int q = 0; q < 32; ++q, at[(q + 3) & 3] += ld4) *at[q & 3] = v[q];
            }
          } else {
#pragma unroll
            for (int q = 0; q < 32; ++q, p += ld) {
              if (c + q >= cols) break;
              if (add) red_add(p, v[q]);
              else *p = v[q];
            }
          }
        }
        add = true;
        tc::fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(in_leader(acc_free + 8 * buf));
        buf ^= 1;
        if (buf == 0) bph ^= 1;
      }
    }
  } else {
    // this thread's group of 32 columns, and its rows of every CONV_GROUPS-th step
    constexpr int RPT = KS / 8 / CONV_WARPS;
    const int grp = (warp - 8) / CONV_WARPS, r0 = (warp - 8) % CONV_WARPS * 8 + (lane & 7), g = lane >> 3;
    const uint32_t full = codes_full + 8 * grp, src0 = base + O_CODES + grp * C_BYTES;
    const uint8_t* sc0 = smem + O_SCALES + grp * (KS * 4) + g;
    const uint32_t ready0 = in_leader(ready);
    uint32_t cph = 0, s = grp, ph = 0;  // phase of the codes' slot; slot of the step and its phase
    for (int64_t i = grp; i < steps; i += CONV_GROUPS) {
      if (!wait_bar(full, cph, failed)) break;
      cph ^= 1;
      // every read in flight before the first conversion
      uint32_t cw[RPT][2][4], sb[RPT], o[RPT][4][4];
#pragma unroll
      for (int rr = 0; rr < RPT; ++rr) {
        const int kr = r0 + rr * 8 * CONV_WARPS;
        sb[rr] = sc0[kr * 4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(cw[rr][h][0]), "=r"(cw[rr][h][1]), "=r"(cw[rr][h][2]), "=r"(cw[rr][h][3])
                       : "r"(src0 + kr * 128 + (((2 * g + h) ^ (kr & 7)) << 4)));
      }
#pragma unroll
      for (int rr = 0; rr < RPT; ++rr) {
        const uint32_t s2 = sb[rr] << 7 | sb[rr] << 23;  // 2^e as bf16, twice (byte 255: infinity)
        const __nv_bfloat162 sc = *reinterpret_cast<const __nv_bfloat162*>(&s2);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          codes4(cw[rr][q >> 2][q & 3], sc, o[rr][q >> 1][(q & 1) * 2], o[rr][q >> 1][(q & 1) * 2 + 1]);
      }
      __syncwarp();
      if (lane == 0) arrive(codes_free + 8 * grp);
      if (!wait_bar(free + 8 * s, ph ^ 1, failed)) break;
#pragma unroll
      for (int rr = 0; rr < RPT; ++rr) {
        const int kr = r0 + rr * 8 * CONV_WARPS;
        const uint32_t dst = base + O_TILES + s * A_BYTES + (g >> 1) * ATOM + kr * 128;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + ((((g & 1) * 4 + q) ^ (kr & 7)) << 4)),
                       "r"(o[rr][q][0]), "r"(o[rr][q][1]), "r"(o[rr][q][2]), "r"(o[rr][q][3])
                       : "memory");
      }
      tc::fence_async_smem();
      __syncwarp();
      if (lane == 0) arrive_cluster(ready0 + 8 * s);
      s += CONV_GROUPS;
      if (s >= NS) {
        s -= NS;
        ph ^= 1;
      }
    }
  }
  let_next_start();
  if (threadIdx.x == 0) wait_for_last();
  __syncwarp();
  if (warp == 2 || warp == 3) pair_wait();
  __syncthreads();
  // a wait gave up, in whichever warp: what is in flight (copies, those of a warp that has issued all of its own too,
  // and products) ends before the pair parts
  if (threadIdx.x == 0 && *failed) linger();
  __syncwarp();
  pair_arrive();
  pair_wait();
  if (threadIdx.x == 0 && *failed && a.status) *a.status = IFK_ERR_TIMEOUT;
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// What is left when the tiles are summed.  The first `joins` blocks add a cut tile's shares, in the
// order of the rows, 16 output columns a block: a thread has four 16-byte reads of a share in
// flight.  The others add the parts of db, 32 columns a block, or, without parts, delta's few rows.
constexpr int JOIN_COLS = 16;
constexpr int FEW_ROWS = 64;  // up to here a pass over delta of its own would cost more than these reads
__global__ void __launch_bounds__(256)
finish_kernel(const Args a, int joins, const float* sums, int parts, const __nv_bfloat16* delta, int64_t ldd,
              float* db) {
  wait_for_last();
  if ((int)blockIdx.x >= joins) {
    __shared__ float sh[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)(blockIdx.x - joins) * 32 + tx;
    float v = 0.f;
    if (c < a.n_out) {
      if (delta)
        for (int64_t r = ty; r < a.rows; r += 8) v += __bfloat162float(delta[r * ldd + c]);
      else
        for (int p = ty; p < parts; p += 8) v += sums[(int64_t)p * a.n_out + c];
    }
    sh[ty][tx] = v;
    __syncthreads();
    if (ty == 0 && c < a.n_out) {
      v = sh[0][tx];
#pragma unroll
      for (int q = 1; q < 8; ++q) v += sh[q][tx];
      db[c] = a.accumulate ? db[c] + v : v;
    }
    return;
  }
  const Plan& p = a.p;
  constexpr int PER = TN / JOIN_COLS;
  const int64_t t = blockIdx.x / PER, b = t * p.Kt;
  const int w0 = p.owner(b), w1 = p.owner(b + p.Kt - 1);
  if (w0 == w1) return;  // one cluster had it all
  const int tile = p.Tdp + (int)t, o = (int)(blockIdx.x % PER) * JOIN_COLS;
  const int64_t i = (int64_t)(tile % p.Ti) * 2 * TM + (threadIdx.x & 63) * 4;
  const int64_t o0 = (int64_t)(tile / p.Ti) * TN + o;
  constexpr int64_t SLOT = TN * 2 * TM;
  constexpr int N = JOIN_COLS / 4;
  const float* src = a.part + (int64_t)(o + (threadIdx.x >> 6)) * (2 * TM) + (threadIdx.x & 63) * 4;
  const int64_t oq = o0 + (threadIdx.x >> 6);
  if (i >= a.n_in || oq >= a.n_out) return;
  float4 v[N];
#pragma unroll
  for (int q = 0; q < N; ++q)
    v[q] = *reinterpret_cast<const float4*>(src + (2 * w0 + 1) * SLOT + q * 4 * (2 * TM));
  for (int c = w0 + 1; c <= w1; ++c) {
    float4 e[N];
#pragma unroll
    for (int q = 0; q < N; ++q) e[q] = *reinterpret_cast<const float4*>(src + 2 * c * SLOT + q * 4 * (2 * TM));
#pragma unroll
    for (int q = 0; q < N; ++q) {
      v[q].x += e[q].x;
      v[q].y += e[q].y;
      v[q].z += e[q].z;
      v[q].w += e[q].w;
    }
  }
#pragma unroll
  for (int q = 0; q < N; ++q) {
    if (oq + q * 4 >= a.n_out) break;
    float* d = a.dW + (oq + q * 4) * a.ldw + i;
    const float r[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
    if (a.vec_out && !a.accumulate && i + 4 <= a.n_in) {
      *reinterpret_cast<float4*>(d) = v[q];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < a.n_in) d[k] = a.accumulate ? d[k] + r[k] : r[k];
    }
  }
}

// delta as bf16 terms in rows TMA can read: fp32 taken apart by truncation into
// three terms of 8 bits each, whose sum is exact (a value that is not finite is in the
// first term alone); bf16 copied.
__device__ __forceinline__ void split3(float x, float (&t)[3]) {
  const uint32_t b = __float_as_uint(x);
  if ((b & 0x7f800000u) == 0x7f800000u) {
    t[0] = (b & 0x007fffffu) ? __uint_as_float(0x7fc00000u) : x;
    t[1] = t[2] = 0.f;
    return;
  }
  t[0] = __uint_as_float(b & 0xffff0000u);
  const float r = x - t[0];
  t[1] = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  t[2] = r - t[1];
}

// One pass over delta before the products, by blocks of 32 V columns, V a lane, over a share of the
// rows: a warp takes every eighth row of the share, four at a time.  part: the shares' column sums (db;
// the warps' sums are added in order), or null.  TERMS: delta's bf16 terms go to `out` (rows x ldo
// each, 16-byte aligned rows, columns past n as 0).
template <typename TD, int V, bool TERMS>
__global__ void __launch_bounds__(256)
delta_pass_kernel(const TD* d, int64_t ldd, int64_t rows, int n, float* part, __nv_bfloat16* out, int64_t ldo) {
  __shared__ float sum[32 * V];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 * V + lane * V;
  float s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.f;
  const int64_t stride = (int64_t)gridDim.y * 8;
  for (int64_t r = (int64_t)blockIdx.y * 8 + wp; r < rows; r += 4 * stride) {
    Raw<TD, V> q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      memset(&q[j], 0, sizeof(q[j]));
      if (r + j * stride < rows) q[j] = load_raw<TD, V>(d + (r + j * stride) * ldd, c, n);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v[V];
      unpack(q[j], v);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += v[i];
      if (TERMS && r + j * stride < rows && c < ldo) {
        __nv_bfloat16* o = out + (r + j * stride) * ldo + c;
        if constexpr (sizeof(TD) == 2) {
          static_assert(!TERMS || V == 1, "rows aligned for more are read in place");
          store_vec<V, true>(o, 0, V, v);
        } else {
          float t[3][V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float e[3];
            split3(v[i], e);
            t[0][i] = e[0];
            t[1][i] = e[1];
            t[2][i] = e[2];
          }
#pragma unroll
          for (int k = 0; k < 3; ++k) store_vec<V, true>(o + k * rows * ldo, 0, V, t[k]);
        }
      }
    }
  }
  let_next_start();
  if (!part) return;
  for (int q = 0; q < 8; ++q) {
    __syncthreads();
    if (q != wp) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) sum[lane * V + i] = q == 0 ? s[i] : sum[lane * V + i] + s[i];
  }
  __syncthreads();
  for (int k = threadIdx.x; k < 32 * V; k += 256) {
    const int cc = blockIdx.x * 32 * V + k;
    if (cc < n) part[(int64_t)blockIdx.y * n + cc] = sum[k];
  }
}

// Shares of the rows: enough blocks of 256 columns to fill the GPU four times, 64 rows a share at least.
int64_t sum_splits(int64_t rows, int64_t n) {
  return std::max<int64_t>(1, std::min<int64_t>(cdiv(rows, 64), SM_COUNT * 4 / cdiv(n, 256)));
}

template <typename TD, int V, bool TERMS>
void delta_pass(const TD* d, int64_t ldd, int64_t rows, int64_t n, int64_t splits, float* part, __nv_bfloat16* out,
                int64_t ldo, cudaStream_t s) {
  delta_pass_kernel<TD, V, TERMS><<<dim3((unsigned)cdiv(TERMS ? ldo : n, 32 * V), (unsigned)splits), 256, 0, s>>>(
      d, ldd, rows, (int)n, part, out, ldo);
}
// fp32 in three terms, or the bf16 rows that TMA cannot read, which are those that are not aligned for 16 bytes.
void copy_delta(const float* d, int64_t ldd, int64_t rows, int64_t n, int64_t splits, float* part, __nv_bfloat16* out,
                int64_t ldo, cudaStream_t s) {
  if (rows_allow<float>(d, ldd, 4)) delta_pass<float, 4, true>(d, ldd, rows, n, splits, part, out, ldo, s);
  else delta_pass<float, 1, true>(d, ldd, rows, n, splits, part, out, ldo, s);
}
void copy_delta(const __nv_bfloat16* d, int64_t ldd, int64_t rows, int64_t n, int64_t splits, float* part,
                __nv_bfloat16* out, int64_t ldo, cudaStream_t s) {
  delta_pass<__nv_bfloat16, 1, true>(d, ldd, rows, n, splits, part, out, ldo, s);
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// Host side of one call: sizes of the workspace parts and the division of the work.
struct Layout {
  bool copy;           // the products read delta's terms in the workspace, not delta
  int terms;
  int64_t ldo;         // pitch of the copied terms
  size_t sums, terms_b, part;
};

Plan make_plan(int64_t rows, int64_t n_out, int64_t n_in, int terms) {
  Plan p;
  p.Ti = (int)cdiv(n_in, TM * 2);
  p.To = (int)cdiv(n_out, TN);
  p.Kt = (int)cdiv(rows, KS) * terms;
  const int64_t T = (int64_t)p.Ti * p.To;
  const int most = CLUSTERS;
  p.Tdp = (int)(T / most * most);
  p.total = (T - p.Tdp) * p.Kt;
  // shares of at least MIN_STEPS steps, or of whole tiles
  p.Gs = (int)mx<int64_t>(1, mn<int64_t>(most, mx<int64_t>(T - p.Tdp, p.total / MIN_STEPS)));
  p.G = p.Tdp ? most : p.Gs;
  return p;
}

Layout layout(int64_t rows, int64_t n_out, int64_t n_in, int dtype, bool copy) {
  Layout l;
  l.terms = dtype == IFK_F32 ? 3 : 1;
  l.copy = copy || dtype == IFK_F32;  // three terms, or rows that TMA cannot read
  l.ldo = cdiv(n_out, 8) * 8;
  l.sums = up256((size_t)sum_splits(rows, n_out) * (size_t)n_out * sizeof(float));
  l.terms_b = l.copy ? up256((size_t)l.terms * (size_t)rows * (size_t)l.ldo * 2) : 0;
  const Plan p = make_plan(rows, n_out, n_in, l.terms);
  l.part = p.total ? (size_t)2 * p.Gs * TN * 2 * TM * sizeof(float) : 0;
  return l;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (EncodeFn)f;
  }();
  return fn;
}

// delta's terms in boxes of 64 columns (128 bytes) x KS rows.  whole: blocks of 64 columns
// are a dimension of their own, and a box has the two that a CTA takes; otherwise (a ragged
// last block) a box has one, and columns past n read as 0.
bool delta_map(CUtensorMap* m, const void* d, int64_t ld, int64_t rows, int64_t n, int terms, bool whole) {
  const cuuint64_t pitch = (cuuint64_t)ld * 2;
  const cuuint64_t dims[4] = {whole ? 64 : (cuuint64_t)n, (cuuint64_t)rows, whole ? (cuuint64_t)n / 64 : 1,
                              (cuuint64_t)terms};
  const cuuint64_t strides[3] = {pitch, whole ? 128 : pitch * (cuuint64_t)rows, pitch * (cuuint64_t)rows};
  const cuuint32_t box[4] = {64, KS, whole ? 2u : 1u, 1}, one[4] = {1, 1, 1, 1};
  return encoder()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(d), dims, strides, box, one,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool codes_map(CUtensorMap* m, const int8_t* c, int64_t ld, int64_t rows, int64_t n) {
  const cuuint64_t dims[2] = {(cuuint64_t)q8::pitch(n), (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {TM, KS}, one[2] = {1, 1};
  return encoder()(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(c), dims, strides, box, one,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch(const CUtensorMap& dm, const CUtensorMap& cm, const Args& a, const float* sums, int parts,
           const __nv_bfloat16* delta, int64_t ldd, float* db, bool behind, cudaStream_t s) {
  static thread_local int done_dev = -1;
  int dev = 0;
  IFK_CUDA_TRY(cudaGetDevice(&dev));
  if (done_dev != dev) {
    IFK_CUDA_TRY(cudaFuncSetAttribute(wgrad_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM));
    done_dev = dev;
  }
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.p.G * 2));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cfg.attrs = behind ? at : at + 1;
  cfg.numAttrs = behind ? 2 : 1;
  IFK_CUDA_TRY(cudaLaunchKernelEx(&cfg, wgrad_kernel, dm, cm, a));
  // no tile is cut when the rest divides into whole tiles
  const int64_t rest = a.p.total / a.p.Kt, joins = rest % a.p.Gs ? rest * (TN / JOIN_COLS) : 0;
  const int64_t blocks = joins + (db ? cdiv(a.n_out, 32) : 0);
  if (blocks) {
    // behind the products' launch only without shares to join: one row of 2048 x 8192 23 -> 20.5 us, but with
    // them (1001 x 521 x 1030 fp32) 31 -> 35 us
    cudaLaunchConfig_t fin{};
    fin.gridDim = dim3((unsigned)blocks);
    fin.blockDim = dim3(256);
    fin.stream = s;
    fin.attrs = at;
    fin.numAttrs = joins ? 0 : 1;
    IFK_CUDA_TRY(cudaLaunchKernelEx(&fin, finish_kernel, a, (int)joins, sums, parts, delta, ldd, db));
  }
  return IFK_OK;
}

template <typename TD>
int run(const TD* delta, int64_t ldd, const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds,
        int64_t rows, int64_t n_out, int64_t n_in, float* dW, int64_t ldw, float* db, int accumulate, int* status,
        uint8_t* ws, bool withhold, cudaStream_t s) {
  if (!encoder()) return IFK_ERR_CUDA;
  const int dtype = sizeof(TD) == 2 ? IFK_BF16 : IFK_F32;
  const Layout l = layout(rows, n_out, n_in, dtype, !rows_allow<TD>(delta, ldd, 8));
  float* sums = (float*)ws;
  __nv_bfloat16* terms = (__nv_bfloat16*)(ws + l.sums);
  Args a;
  a.p = make_plan(rows, n_out, n_in, l.terms);
  a.terms = l.terms;
  a.scales = scales;
  a.lds = lds;
  a.rows = rows;
  a.n_out = n_out;
  a.n_in = n_in;
  a.ldw = ldw;
  a.dW = dW;
  a.part = (float*)(ws + l.sums + l.terms_b);
  a.accumulate = accumulate;
  a.vec_out = ((uintptr_t)dW & 15) == 0 && ldw % 4 == 0;
  a.vec_scales = ((uintptr_t)scales & 3) == 0 && lds % 4 == 0;
  a.status = status;
  a.withhold = withhold;
  a.copied = l.copy;
  const int parts = (int)sum_splits(rows, n_out);
  const bool pass = l.copy || (db && rows > FEW_ROWS);
  const void* src = delta;
  int64_t ld = ldd;
  if (l.copy) {
    copy_delta(delta, ldd, rows, n_out, parts, db ? sums : nullptr, terms, l.ldo, s);
    IFK_CUDA_TRY(cudaGetLastError());
    src = terms;
    ld = l.ldo;
  } else if (pass) {
    if constexpr (sizeof(TD) == 2) delta_pass<TD, 8, false>(delta, ldd, rows, n_out, parts, sums, nullptr, 0, s);
    IFK_CUDA_TRY(cudaGetLastError());
  }
  CUtensorMap dm, cm;
  a.whole = n_out % 64 == 0;
  if (!delta_map(&dm, src, ld, rows, n_out, l.terms, a.whole) || !codes_map(&cm, codes, ldc, rows, n_in))
    return IFK_ERR_SHAPE;
  const bool few = !l.copy && rows <= FEW_ROWS;  // delta is bf16 then
  return launch(dm, cm, a, sums, parts, few ? (const __nv_bfloat16*)(const void*)delta : nullptr, ldd, db, pass, s);
}

}  // namespace

size_t q8_wgrad_bytes(int64_t rows, int64_t n_out, int64_t n_in, int dtype, bool copy) {
  const Layout l = layout(rows, n_out, n_in, dtype, copy);
  return l.sums + l.terms_b + l.part;
}

int q8_wgrad_run(const void* delta, int64_t ldd, int dtype, const int8_t* codes, int64_t ldc, const uint8_t* scales,
                 int64_t lds, int64_t rows, int64_t n_out, int64_t n_in, float* dW, int64_t ldw, float* db,
                 int accumulate, int* status, uint8_t* ws, bool withhold, cudaStream_t s) {
  if (dtype == IFK_F32)
    return run((const float*)delta, ldd, codes, ldc, scales, lds, rows, n_out, n_in, dW, ldw, db, accumulate, status,
               ws, withhold, s);
  return run((const __nv_bfloat16*)delta, ldd, codes, ldc, scales, lds, rows, n_out, n_in, dW, ldw, db, accumulate,
             status, ws, withhold, s);
}

}  // namespace ifk
