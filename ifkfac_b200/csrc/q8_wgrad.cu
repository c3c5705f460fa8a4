// Weight and bias gradient of a linear layer from its 8-bit input rows
// (ifk_q8_wgrad): dW = delta^T X, db = column sums of delta.
//
// dW is a matrix product whose long axis is the rows, so both operands are
// M/N-major: a row of delta or of X is contiguous along the output.  The 8-bit
// rows take the M side (128 input columns a CTA), delta the N side (256 output
// columns), so the accumulator in TMEM has an input column a lane and the
// epilogue's stores are contiguous along dW's rows.
//
// Per step of 64 rows, TMA brings delta (bf16, 128-byte swizzle) and the codes
// into a stage; eight warps turn the codes into bf16 in the same layout; one
// thread issues the four tcgen05.mma of the step.  A code times its power-of-two
// scale is exact in bf16, so the products are exact and only the fp32 sums round.
// An fp32 delta is taken apart beforehand into three bf16 terms (8 + 8 + 8 bits,
// by truncation: exact), and each 64 rows take three steps.
//
// With CG = 2 a pair of CTAs shares one 256 x 256 tile (tcgen05 cta_group::2): each
// converts its own 128 input columns and loads half of delta's columns.
//
// The tensor core truncates as it adds to the accumulator, so a long sum drifts
// towards zero by about 7e-9 of itself a tcgen05.mma; after CHUNK steps (120 of them)
// the accumulator is therefore added to dW in L2 (red.global.add, rounded to nearest;
// one thread owns an element, so the order is fixed) while the next chunk goes to the
// other half of TMEM.
//
// Work: whole waves of tiles first, every cluster a tile at a time; the tiles that
// are left over are cut along the rows into equal shares for all clusters.  A share
// that is not a whole tile goes to the workspace, and a second kernel adds a
// tile's shares in order.
#include <cuda.h>

#include "q8.cuh"
#include "ifk_internal.h"
#include "tc.cuh"

namespace ifk {

namespace {

constexpr int KS = 64;        // rows a step
constexpr int TM = 128;       // input columns a CTA
constexpr int TN = 256;       // output columns a tile
constexpr int CHUNK = 30;     // steps a TMEM accumulator sums: 30 row blocks, or 10 in three terms
constexpr int CONV_WARPS = 4; // a step's converting warps; two such groups take turns
constexpr int THREADS = 512;  // warps: 0 TMA, 1 MMA, 2 TMEM, 3 scales, 4-7 epilogue, 8-15 conversion
constexpr int AHEAD = 4;      // steps the scales are loaded ahead
constexpr uint32_t A_BYTES = TM * KS * 2, C_BYTES = TM * KS;
constexpr uint32_t ATOM = 64 * KS * 2;  // 64 columns (128 bytes) of KS rows
constexpr int SM_COUNT = 148;
constexpr int MIN_STEPS = 4;  // least steps a share of a cut tile is worth

template <int CG>
struct Cfg {
  static constexpr uint32_t B_BYTES = TN / CG * KS * 2;
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES + C_BYTES;
  static constexpr int STAGES = CG == 2 ? 5 : 4;
  static constexpr uint32_t SCALES = STAGES * STAGE;  // per stage KS x 4 bytes
  static constexpr uint32_t BARS = SCALES + STAGES * KS * 4;
  static constexpr uint32_t SMEM = BARS + (3 * STAGES + 4) * 8 + 16;
};

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
  float* part;         // [2 Gs][TN][CG TM]
  int accumulate;
  bool vec_scales;     // rows of scales start at multiples of 4 bytes
  int* status;
};

// Step k of a tile: which block of KS rows, and which of delta's terms.  The terms of
// a chunk's rows come smallest first, so that the sums of the small ones are truncated
// at their own size.
struct Step {
  int block, term;
};
__device__ __forceinline__ Step step_at(const Args& a, int k) {
  if (a.terms == 1) return {k, 0};
  const int sup = k / CHUNK, rem = k - sup * CHUNK;
  const int nb = mn(CHUNK / 3, a.p.Kt / 3 - sup * (CHUNK / 3));
  const int q = rem / nb;
  return {sup * (CHUNK / 3) + rem - q * nb, 2 - q};
}
// End of the chunk that step k is in.
__device__ __forceinline__ int chunk_end(int k, int k1) { return mn((k / CHUNK + 1) * CHUNK, k1); }

// One piece of work: steps k0 .. k1 of a tile; slot < 0: the whole tile.
struct Piece {
  int tile, k0, k1, slot;
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

__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// Bounded wait: gives up after two seconds, or when another warp of the CTA has.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int* failed) {
  uint64_t t0 = 0;
  for (uint32_t it = 0;; ++it) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if ((it & 63) == 63) {
      if (*failed) return false;
      const uint64_t t = now_ns();
      if (t0 == 0) t0 = t;
      else if (t - t0 > 2000000000ull) {
        *failed = 1;
        return false;
      }
    }
  }
}

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Arrive on the barrier at the same offset in the cluster's first CTA.
template <int CG>
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
  if (CG == 1) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .b32 ra;\n\t"
        "mapa.shared::cluster.u32 ra, %0, 0;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [ra];\n\t}\n" ::"r"(bar)
        : "memory");
  }
}

// Operand tiles: M/N-major, 128-byte swizzle.  64 columns of 8 rows are one 1024-byte
// atom; the next 8 rows follow at SBO = 1024 bytes, the next 64 columns at LBO = ATOM.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(ATOM >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  if (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
        : "memory");
}

// Arrive on this barrier (in both CTAs of a pair) when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void alloc_tmem(uint32_t slot) {
  if (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void free_tmem(uint32_t base) {
  if (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(base) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(base) : "memory");
}

template <int CG>
__device__ __forceinline__ void sync_cluster() {
  if (CG == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
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

template <int CG>
__global__ void __launch_bounds__(THREADS, 1)
wgrad_kernel(const __grid_constant__ CUtensorMap dmap, const __grid_constant__ CUtensorMap cmap, const Args a) {
  using C = Cfg<CG>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = tc::smem_u32(smem);
  const uint32_t full = base + C::BARS, ready = full + 8 * C::STAGES, empty = ready + 8 * C::STAGES;
  const uint32_t acc_full = empty + 8 * C::STAGES, acc_empty = acc_full + 16;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + C::BARS + (3 * C::STAGES + 4) * 8);
  volatile int* failed = reinterpret_cast<volatile int*>(slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? (blockIdx.x & 1) : 0;
  const int cluster = blockIdx.x / CG;

  if (threadIdx.x == 0) {
    *failed = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      tc::mbar_init(reinterpret_cast<uint64_t*>(smem + C::BARS) + s, 2);  // the copies and the scales
      tc::mbar_init(reinterpret_cast<uint64_t*>(smem + C::BARS) + C::STAGES + s, CONV_WARPS * CG);
      tc::mbar_init(reinterpret_cast<uint64_t*>(smem + C::BARS) + 2 * C::STAGES + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(reinterpret_cast<uint64_t*>(smem + C::BARS) + 3 * C::STAGES + b, 1);
      tc::mbar_init(reinterpret_cast<uint64_t*>(smem + C::BARS) + 3 * C::STAGES + 2 + b, 4 * CG);
    }
  }
  if (warp == 2) alloc_tmem<CG>(tc::smem_u32(slot));
  tc::fence_before();
  __syncthreads();
  sync_cluster<CG>();
  tc::fence_after();
  const uint32_t tmem = *slot;

  Walk walk(a.p, cluster);
  Piece w;
  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      while (ok && walk.next(w)) {
        const int ti = w.tile % a.p.Ti, to = w.tile / a.p.Ti;
        const int x = (ti * CG + (int)rank) * TM, o = to * TN + (int)rank * (TN / CG);
        for (int k = w.k0; k < w.k1; ++k, ++it) {
          const uint32_t s = it % C::STAGES, ph = it / C::STAGES & 1;
          if (!wait_bar(empty + 8 * s, ph ^ 1, failed)) {
            ok = false;
            break;
          }
          const uint32_t st = base + s * C::STAGE, bar = full + 8 * s;
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(C::B_BYTES + C_BYTES)
                       : "memory");
          const Step sp = step_at(a, k);
          const int row = sp.block * KS;
          tma_2d(st + A_BYTES + C::B_BYTES, &cmap, x, row, bar);
#pragma unroll
          for (int j = 0; j < TN / CG / 64; ++j)
            tma_3d(st + A_BYTES + j * ATOM, &dmap, o + j * 64, row, sp.term, bar);
        }
      }
      // leave with no copy in flight (the last STAGES steps'); after a failed wait too
      for (uint32_t q = it > C::STAGES ? it - C::STAGES : 0; q < it; ++q) {
        int quiet = 0;
        if (!wait_bar(full + 8 * (q % C::STAGES), q / C::STAGES & 1, &quiet)) break;
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc = tc::idesc_bf16(TM * CG, TN, true, true);
      uint32_t it = 0, buf = 0, bph = 0;
      bool ok = true;
      while (ok && walk.next(w)) {
        for (int c0 = w.k0, c1; ok && c0 < w.k1; c0 = c1) {
          c1 = chunk_end(c0, w.k1);
          if (!wait_bar(acc_empty + 8 * buf, bph ^ 1, failed)) {
            ok = false;
            break;
          }
          tc::fence_after();
          for (int k = c0; k < c1; ++k, ++it) {
            const uint32_t s = it % C::STAGES, ph = it / C::STAGES & 1;
            if (!wait_bar(ready + 8 * s, ph, failed)) {
              ok = false;
              break;
            }
            tc::fence_after();
            const uint64_t ad = desc_sw128(base + s * C::STAGE), bd = desc_sw128(base + s * C::STAGE + A_BYTES);
#pragma unroll
            for (int j = 0; j < KS / 16; ++j)
              mma<CG>(tmem + buf * TN, ad + tc::doff(j * 2048), bd + tc::doff(j * 2048), idesc,
                      (k > c0 || j > 0) ? 1u : 0u);
            commit<CG>(empty + 8 * s);
          }
          commit<CG>(acc_full + 8 * buf);
          if (!ok) {
            // a wait gave up: leave once the products already issued are done
            int quiet = 0;
            wait_bar(acc_full + 8 * buf, bph, &quiet);
          }
          buf ^= 1;
          if (buf == 0) bph ^= 1;
        }
      }
    }
  } else if (warp == 3) {
    // the scale bytes of a stage: rows lane and lane + 32, four groups each, loaded AHEAD steps early
    uint32_t it = 0;
    bool ok = true;
    const int64_t groups = q8::pitch(a.n_in) / q8::GROUP;
    while (ok && walk.next(w)) {
      const int64_t gi = (int64_t)(w.tile % a.p.Ti * CG + (int)rank) * (TM / q8::GROUP);
      const bool vec = a.vec_scales && gi + 4 <= groups;
      auto load = [&](int k, int h) -> uint32_t {
        if (k >= w.k1) return 0u;
        const int64_t r = (int64_t)step_at(a, k).block * KS + h * 32 + lane;
        if (r >= a.rows) return 0u;
        const uint8_t* p = a.scales + r * a.lds + gi;
        if (vec) return *reinterpret_cast<const uint32_t*>(p);
        uint32_t v = 0;
        for (int g = 0; g < 4; ++g)
          if (gi + g < groups) v |= (uint32_t)p[g] << (8 * g);
        return v;
      };
      uint32_t q[AHEAD][2];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        q[j][0] = load(w.k0 + j, 0);
        q[j][1] = load(w.k0 + j, 1);
      }
      for (int k = w.k0; ok && k < w.k1; k += AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          if (!ok || k + j >= w.k1) break;
          const uint32_t s = it % C::STAGES, ph = it / C::STAGES & 1;
          if (!wait_bar(empty + 8 * s, ph ^ 1, failed)) {
            ok = false;
            break;
          }
          uint32_t* d = reinterpret_cast<uint32_t*>(smem + C::SCALES + s * (KS * 4));
          d[lane] = q[j][0];
          d[32 + lane] = q[j][1];
          q[j][0] = load(k + j + AHEAD, 0);
          q[j][1] = load(k + j + AHEAD, 1);
          __syncwarp();
          if (lane == 0)
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(full + 8 * s) : "memory");
          ++it;
        }
      }
    }
  } else if (warp >= 4 && warp < 8) {
    uint32_t buf = 0, bph = 0;
    const int wq = warp & 3;  // the quarter of TMEM's lanes this warp reads
    bool ok = true;
    while (ok && walk.next(w)) {
      const int ti = w.tile % a.p.Ti, to = w.tile / a.p.Ti;
      const int m = (int)rank * TM + wq * 32 + lane;
      const int64_t i = (int64_t)ti * CG * TM + m, o0 = (int64_t)to * TN;
      // where this thread's column of the tile goes: dW, or its share's slot
      const bool to_part = w.slot >= 0;
      float* d = to_part ? a.part + (int64_t)w.slot * (TN * CG * TM) + m : a.dW + o0 * a.ldw + i;
      const int64_t ld = to_part ? CG * TM : a.ldw;
      const int cols = to_part ? TN : (i < a.n_in ? (int)mn<int64_t>(TN, a.n_out - o0) : 0);
      bool add = !to_part && a.accumulate;
      for (int c0 = w.k0; c0 < w.k1; c0 = chunk_end(c0, w.k1)) {
        if (!wait_bar(acc_full + 8 * buf, bph, failed)) {
          ok = false;
          break;
        }
        tc::fence_after();
        for (int c = 0; c < TN; c += 32) {
          float v[32];
          tc::tmem_ld32(tmem + buf * TN + c + ((uint32_t)(wq * 32) << 16), v);
          float* p = d + c * ld;
          if (c + 32 <= cols) {
            if (add) {
#pragma unroll
              for (int q = 0; q < 32; ++q, p += ld) asm volatile("red.global.add.f32 [%0], %1;" ::"l"(p), "f"(v[q]) : "memory");
            } else {
#pragma unroll
              for (int q = 0; q < 32; ++q, p += ld) *p = v[q];
            }
          } else {
#pragma unroll
            for (int q = 0; q < 32; ++q, p += ld)
              if (c + q < cols) {
                if (add) asm volatile("red.global.add.f32 [%0], %1;" ::"l"(p), "f"(v[q]) : "memory");
                else *p = v[q];
              }
          }
        }
        add = true;
        tc::fence_before();
        __syncwarp();
        if (lane == 0) arrive_leader<CG>(acc_empty + 8 * buf);
        buf ^= 1;
        if (buf == 0) bph ^= 1;
      }
    }
  } else if (warp >= 8) {
    // this thread's group of 32 columns and its two rows of every other step
    const int grp = (warp - 8) / CONV_WARPS, r0 = (warp - 8) % CONV_WARPS * 8 + (lane & 7), g = lane >> 3;
    uint32_t it = 0;
    bool ok = true;
    while (ok && walk.next(w)) {
      const uint32_t end = it + (uint32_t)(w.k1 - w.k0);
      for (; it < end; ++it) {
        if ((int)(it & 1) != grp) continue;
        const uint32_t s = it % C::STAGES, ph = it / C::STAGES & 1;
        if (!wait_bar(full + 8 * s, ph, failed)) {
          ok = false;
          break;
        }
        const uint32_t st = base + s * C::STAGE;
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const int kr = r0 + rr * 32;
          const uint32_t src = st + A_BYTES + C::B_BYTES + kr * 128;
          const uint32_t dst = st + (g >> 1) * ATOM + kr * 128;
          const uint32_t s0 = smem[C::SCALES + s * (KS * 4) + kr * 4 + g];
          const uint32_t sb = s0 << 7 | s0 << 23;  // 2^e as bf16, twice (byte 255: infinity)
          const __nv_bfloat162 sc = *reinterpret_cast<const __nv_bfloat162*>(&sb);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t cw[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(cw[0]), "=r"(cw[1]), "=r"(cw[2]), "=r"(cw[3])
                         : "r"(src + (((2 * g + h) ^ (kr & 7)) << 4)));
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t o[4];
              codes4(cw[2 * q], sc, o[0], o[1]);
              codes4(cw[2 * q + 1], sc, o[2], o[3]);
              asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                               dst + ((((g & 1) * 4 + h * 2 + q) ^ (kr & 7)) << 4)),
                           "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3])
                           : "memory");
            }
          }
        }
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) arrive_leader<CG>(ready + 8 * s);
      }
    }
  }
  __syncwarp();
  __syncthreads();
  sync_cluster<CG>();
  if (threadIdx.x == 0 && *failed && a.status) *a.status = IFK_ERR_TIMEOUT;
  if (warp == 2) free_tmem<CG>(tmem);
}

// A cut tile's shares, added in the order of the rows.  A block takes 16 output columns.
template <int CG>
__global__ void __launch_bounds__(CG * TM) join_kernel(const Args a) {
  const Plan& p = a.p;
  const int64_t t = blockIdx.x, b = t * p.Kt;
  const int w0 = p.owner(b), w1 = p.owner(b + p.Kt - 1);
  if (w0 == w1) return;  // one cluster had it all
  const int tile = p.Tdp + (int)t;
  const int64_t i = (int64_t)(tile % p.Ti) * CG * TM + threadIdx.x;
  const int64_t o0 = (int64_t)(tile / p.Ti) * TN + blockIdx.y * 16;
  if (i >= a.n_in) return;
  constexpr int64_t SLOT = TN * CG * TM;
  const float* src = a.part + (int64_t)blockIdx.y * 16 * (CG * TM) + threadIdx.x;
#pragma unroll 4
  for (int q = 0; q < 16; ++q) {
    if (o0 + q >= a.n_out) break;
    const float* s = src + q * (CG * TM);
    float v = s[(2 * w0 + 1) * SLOT];
    for (int c = w0 + 1; c <= w1; ++c) v += s[2 * c * SLOT];
    float* d = a.dW + (o0 + q) * a.ldw + i;
    *d = a.accumulate ? *d + v : v;
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

template <typename TD>
__global__ void __launch_bounds__(256) terms_kernel(const TD* delta, int64_t ldd, bool vec, int64_t rows, int64_t n,
                                                    __nv_bfloat16* out, int64_t ldo) {
  const int64_t upr = ldo / 8, total = rows * upr;
  for (int64_t u = blockIdx.x * 256ll + threadIdx.x; u < total; u += gridDim.x * 256ll) {
    const int64_t r = u / upr, c = (u - r * upr) * 8;
    float v[8];
    load8(delta + r * ldd, c, n, vec, v);
    __nv_bfloat16* d = out + r * ldo;
    if (sizeof(TD) == 2) {
      store8(d, c, ldo, true, v);
    } else {
      float t[3][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float e[3];
        split3(v[i], e);
        t[0][i] = e[0];
        t[1][i] = e[1];
        t[2][i] = e[2];
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) store8(d + q * rows * ldo, c, ldo, true, t[q]);
    }
  }
}

// Sums over a share of the rows of 256 columns, 8 a lane; warps take every eighth row
// of the share and are added in order.
template <typename TD>
__global__ void __launch_bounds__(256)
column_sums_kernel(const TD* d, int64_t ldd, bool vec, int64_t rows, int64_t n, float* part) {
  __shared__ float sum[256];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 256 + lane * 8;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t r = (int64_t)blockIdx.y * 8 + wp; r < rows; r += (int64_t)gridDim.y * 8) {
    float v[8];
    load8(d + r * ldd, c, n, vec, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] += v[i];
  }
  for (int q = 0; q < 8; ++q) {
    __syncthreads();
    if (q != wp) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[lane * 8 + i] = q == 0 ? s[i] : sum[lane * 8 + i] + s[i];
  }
  __syncthreads();
  const int64_t cc = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (cc < n) part[(int64_t)blockIdx.y * n + cc] = sum[threadIdx.x];
}

int64_t sum_splits(int64_t rows, int64_t n) {
  return mx<int64_t>(1, mn<int64_t>(cdiv(rows, 64), 148 * 4 / cdiv(n, 256)));
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// Host side of one call: sizes of the workspace parts and the division of the work.
struct Layout {
  bool copy;           // delta goes through terms_kernel
  int terms;
  int64_t ldo;         // pitch of the copied terms
  size_t sums, terms_b, part;
};

constexpr int CG_USED = 2;

Plan make_plan(int64_t rows, int64_t n_out, int64_t n_in, int terms) {
  Plan p;
  p.Ti = (int)cdiv(n_in, TM * CG_USED);
  p.To = (int)cdiv(n_out, TN);
  p.Kt = (int)cdiv(rows, KS) * terms;
  const int64_t T = (int64_t)p.Ti * p.To;
  const int most = SM_COUNT / CG_USED;
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
  l.copy = copy || dtype == IFK_F32;
  l.ldo = cdiv(n_out, 8) * 8;
  l.sums = up256((size_t)sum_splits(rows, n_out) * (size_t)n_out * sizeof(float));
  l.terms_b = l.copy ? up256((size_t)l.terms * (size_t)rows * (size_t)l.ldo * 2) : 0;
  const Plan p = make_plan(rows, n_out, n_in, l.terms);
  l.part = p.total ? (size_t)2 * p.Gs * TN * CG_USED * TM * sizeof(float) : 0;
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

// delta's terms: columns, rows, terms; boxes of 64 columns (128 bytes) x KS rows.
bool delta_map(CUtensorMap* m, const void* d, int64_t ld, int64_t rows, int64_t n, int terms) {
  const cuuint64_t dims[3] = {(cuuint64_t)n, (cuuint64_t)rows, (cuuint64_t)terms};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * (cuuint64_t)rows};
  const cuuint32_t box[3] = {64, KS, 1}, one[3] = {1, 1, 1};
  return encoder()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(d), dims, strides, box, one,
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

template <int CG>
int launch(const CUtensorMap& dm, const CUtensorMap& cm, const Args& a, cudaStream_t s) {
  static thread_local int done_dev = -1;
  int dev = 0;
  IFK_CUDA_TRY(cudaGetDevice(&dev));
  if (done_dev != dev) {
    IFK_CUDA_TRY(cudaFuncSetAttribute(wgrad_kernel<CG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)Cfg<CG>::SMEM));
    done_dev = dev;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.p.G * CG));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Cfg<CG>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  IFK_CUDA_TRY(cudaLaunchKernelEx(&cfg, wgrad_kernel<CG>, dm, cm, a));
  if (a.p.total) join_kernel<CG><<<dim3((unsigned)(a.p.total / a.p.Kt), TN / 16), CG * TM, 0, s>>>(a);
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

template <typename TD>
int run(const TD* delta, int64_t ldd, const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds,
        int64_t rows, int64_t n_out, int64_t n_in, float* dW, int64_t ldw, float* db, int accumulate, int* status,
        uint8_t* ws, cudaStream_t s) {
  if (!encoder()) return IFK_ERR_CUDA;
  const int dtype = sizeof(TD) == 2 ? IFK_BF16 : IFK_F32;
  const Layout l = layout(rows, n_out, n_in, dtype, !rows_aligned(delta, ldd));
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
  a.vec_scales = ((uintptr_t)scales & 3) == 0 && lds % 4 == 0;
  a.status = status;
  const void* src = delta;
  int64_t ld = ldd;
  if (l.copy) {
    const int64_t g = cdiv(rows * (l.ldo / 8), 256);
    terms_kernel<TD><<<(unsigned)mn<int64_t>(g, SM_COUNT * 16), 256, 0, s>>>(delta, ldd, rows_aligned(delta, ldd), rows,
                                                                            n_out, terms, l.ldo);
    IFK_CUDA_TRY(cudaGetLastError());
    src = terms;
    ld = l.ldo;
  }
  CUtensorMap dm, cm;
  if (!delta_map(&dm, src, ld, rows, n_out, l.terms) || !codes_map(&cm, codes, ldc, rows, n_in)) return IFK_ERR_SHAPE;
  const int rc = launch<CG_USED>(dm, cm, a, s);
  if (rc != IFK_OK || !db) return rc;
  const int64_t parts = sum_splits(rows, n_out);
  column_sums_kernel<TD><<<dim3((unsigned)cdiv(n_out, 256), (unsigned)parts), 256, 0, s>>>(
      delta, ldd, rows_aligned(delta, ldd), rows, n_out, sums);
  IFK_CUDA_TRY(cudaGetLastError());
  return sum_parts_run(sums, parts, n_out, db, nullptr, nullptr, accumulate, s);
}

}  // namespace

size_t q8_wgrad_bytes(int64_t rows, int64_t n_out, int64_t n_in, int dtype) {
  const Layout l = layout(rows, n_out, n_in, dtype, true);
  return l.sums + l.terms_b + l.part;
}

int q8_wgrad_run(const void* delta, int64_t ldd, int dtype, const int8_t* codes, int64_t ldc, const uint8_t* scales,
                 int64_t lds, int64_t rows, int64_t n_out, int64_t n_in, float* dW, int64_t ldw, float* db,
                 int accumulate, int* status, uint8_t* ws, cudaStream_t s) {
  if (dtype == IFK_F32)
    return run((const float*)delta, ldd, codes, ldc, scales, lds, rows, n_out, n_in, dW, ldw, db, accumulate, status,
               ws, s);
  return run((const __nv_bfloat16*)delta, ldd, codes, ldc, scales, lds, rows, n_out, n_in, dW, ldw, db, accumulate,
             status, ws, s);
}

}  // namespace ifk
