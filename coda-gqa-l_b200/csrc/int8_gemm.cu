// y[m][n] = x_scale[m] * w_scale[n] * sum_k x[m][k] w[n][k]  (+ bias[n]) (+ residual[m][n]), x and w in 8-bit integers.
// The sum is exact in 32 bits (K <= 131071: 2^14 * K < 2^31), the rest is fp32, rounded once to the type of y.  The sum is
// scaled by one factor after the other: the product of both scales may leave fp32's range where the result does not.
//
// Both kernels run tcgen05.mma.kind::i8 with the operands swapped: the WEIGHT rows (output channels) are the MMA's M,
// the tokens its N, so that a decode step's few tokens waste no tensor work, and a thread of the epilogue, which owns a
// TMEM lane, owns a channel: its scale and bias are two registers, and a warp's store of one token is 32 neighbouring
// channels.  Operands come by TMA, 128 bytes of K a row (128-byte swizzle); what lies behind K, M or N reads as zero.
// No load is multicast.  Every wait is bounded (status word, CTA abort word).
#include "coda_common.cuh"
#include "tma_utils.cuh"
#include "tensor_maps.h"
#include <math.h>

namespace {

using tma::smem_u32;

constexpr int IG_BK = 128;                 // bytes of K a stage holds: one swizzle row, four MMAs
constexpr int IG_BN = 128;                 // channels per CTA (MMA M of one CTA)
constexpr int IG_WBOX = IG_BN * IG_BK;
constexpr int IG_MAX_SMEM = 227 * 1024;
// dynamic shared memory of a split CTA that has an SM to itself / shares it with another (1 KB is the system's, 2 KB static)
constexpr int IS_SMEM_WHOLE = 225 * 1024, IS_SMEM_HALF = 111 * 1024;

struct Int8GemmParams {
  int M, N, K, nkb;                        // nkb = ceil(K / 128)
  const float* x_scale; const float* w_scale;
  const void* bias; const void* res; long long res_rs;
  void* y; long long y_rs;
  int* status;
  int ctiles, ttiles;                      // tiles of channels / of tokens
  int group;                               // channel tiles that the pair kernel walks over together
  int w_ready;                             // the weights were complete before an earlier product on this stream began
};

__device__ __forceinline__ bool ig_elect() {
  uint32_t pred;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void ig_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ig_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ig_wait_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void ig_next_grid() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void ig_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void ig_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t ig_mapa(uint32_t local, int rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ void ig_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void ig_ld8(uint32_t taddr, int (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// K-major operand, rows of 128 bytes with the 128-byte swizzle, 8-row groups 1024 bytes apart, descriptor version 1
__device__ __forceinline__ uint64_t ig_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// 32-bit integer accumulator, signed 8-bit x signed 8-bit, both operands K-major
__device__ __forceinline__ constexpr uint32_t ig_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Four MMAs: 128 bytes of K of one stage
template <int CG>
__device__ __forceinline__ void ig_mma_stage(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool first) {
#pragma unroll
  for (int kk = 0; kk < IG_BK / 32; ++kk) {
    const uint32_t acc = first && kk == 0 ? 0u : 1u;
    if constexpr (CG == 2)
      asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}"
                   ::"r"(d_tmem), "l"(adesc + kk * 2), "l"(bdesc + kk * 2), "r"(idesc), "r"(acc) : "memory");
    else
      asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}"
                   ::"r"(d_tmem), "l"(adesc + kk * 2), "l"(bdesc + kk * 2), "r"(idesc), "r"(acc) : "memory");
  }
}
// One thread waits (addresses are shared-memory ones); the bounded loop behind the first poll is out of line, so that the
// issuing loops stay short.  Acquires at cluster scope: the pair kernel's barriers are arrived at from the other CTA too.
__device__ __forceinline__ uint32_t ig_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok;
}
__device__ __noinline__ void ig_wait_slow(uint32_t bar, uint32_t parity, int* status, int code, int* abort, int limit) {
  for (int it = 0; it < limit; ++it) {
    if (ig_try(bar, parity)) return;
    if ((it & 15) == 15 && *reinterpret_cast<volatile int*>(abort) != 0) return;
  }
  *reinterpret_cast<volatile int*>(abort) = code;
  if (status) atomicCAS(status, 0, code);
}
__device__ __forceinline__ void ig_wait(uint32_t bar, uint32_t parity, int* status, int code, int* abort, int limit = tma::WAIT_LIMIT) {
  if (!ig_try(bar, parity)) ig_wait_slow(bar, parity, status, code, abort, limit);
}
// The converged warp waits: one lane polls.
__device__ __forceinline__ void ig_wait_warp(uint32_t bar, uint32_t parity, int* status, int code, int* abort) {
  if (ig_elect()) ig_wait(bar, parity, status, code, abort);
  __syncwarp();
}
__device__ __forceinline__ void ig_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A CTA whose bounded wait gave up leaves its copies time to land before it returns its shared memory.
__device__ __forceinline__ void ig_settle(const int* abortw) {
  if (*reinterpret_cast<const volatile int*>(abortw) != 0)
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
}

// ---- few tokens: a stream of the weights --------------------------------------------------------------
// With few tokens the product is one pass over the weights, bound by HBM: what counts is that every SM loads its share.
// A tile is 128 channels by NT tokens, and the S CTAs of a cluster take equal runs of its K.  The partial sums are integers:
// any order gives the same bits.  They meet through distributed shared memory, each CTA finishing `per` of the tokens.
// Back to back on cold weights: 32 x 4096 -> 6177 9.1 us, 1 x 512 -> 777 2.5 us; what grows with the size does so at the HBM's
// rate (8192 x 8192 weights 13.2 us, 4096 x 4096 6.1: 50 MB in 7.1 us), some 3.5 us do not.
// Warp 0 = TMA producer, warp 1 = MMA issuer and TMEM owner, warps 2-5 = epilogue; residual and scales of the epilogue are
// in shared memory before the last MMA is done.
constexpr int IS_THREADS = 192, IS_KPS = 2, IS_MAX_STAGES = 8;
static_assert((IS_SMEM_WHOLE - 1024) / (IS_KPS * (IG_BN + 16) * IG_BK) <= IS_MAX_STAGES, "more stages than barriers");

struct SplitShape {
  int split, per;                          // CTAs per cluster, tokens a CTA finishes (a multiple of 8)
  int stages, ring, res, xch, total;       // stages of the ring; bytes of ring, residual tile, exchange, everything
  int flat;                                // K is no multiple of 128: a box holds one k-block, not IS_KPS
};

template <typename T, int NT>
__global__ void __launch_bounds__(IS_THREADS)
int8_split_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, Int8GemmParams p, SplitShape h) {
  constexpr uint32_t COLS = NT < 32 ? 32 : NT;
  constexpr int XBOX = NT * IG_BK, STAGE = IS_KPS * (IG_WBOX + XBOX);
  constexpr uint32_t EMPTY = IS_MAX_STAGES * 8;
  extern __shared__ unsigned char is_raw[];
  __shared__ uint64_t full[2 * IS_MAX_STAGES], acc_full;     // a stage's barrier when it is full, and EMPTY bytes on when free
  __shared__ float s_sx[NT];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  unsigned char* smem = is_raw + ((1024u - (smem_u32(is_raw) & 1023u)) & 1023u);
  T* s_res = reinterpret_cast<T*>(smem + h.ring);         // [per][128]
  int* xch = reinterpret_cast<int*>(smem + h.ring + h.res); // [split][per][128]
  int* const abortw = &s_abort;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int S = h.split, rank = S > 1 ? blockIdx.x % S : 0, n0 = (S > 1 ? blockIdx.x / S : blockIdx.x) * IG_BN;
  const int m0 = blockIdx.y * NT, mt = min(NT, p.M - m0);
  const int all = (p.nkb + IS_KPS - 1) / IS_KPS, s0 = all * rank / S, ns = all * (rank + 1) / S - s0;   // stages; what lies behind K is zero

  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < h.stages; ++i) { tma::mbar_init(&full[i], 1); tma::mbar_init(&full[IS_MAX_STAGES + i], 1); }
    tma::mbar_init(&acc_full, 1);
    tma::fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    ig_fence_before();
  }
  __syncthreads();
  ig_fence_after();
  const uint32_t tmem = s_tmem;
  if (S > 1) ig_cluster_arrive();                       // its wait: before anything is sent to another CTA

  const uint32_t ring0 = smem_u32(smem), ring_end = ring0 + h.ring, full0 = smem_u32(&full[0]);
  const int quarter = warp & 3, row = quarter * 32 + lane, n = n0 + row;
  const bool mine = warp >= 2 && n < p.N;
  const int t0 = rank * h.per, nt = max(0, min(mt - t0, h.per));   // tokens this CTA finishes
  float sw = 0.f, bias = 0.f;
  if (warp == 0) {
    if (ig_elect()) {
      // a box of `map`: (byte of K, row, 0) where it is one k-block, else (0, row, k-block)
      auto load = [&](uint32_t to, uint32_t bar, const CUtensorMap* map, int box, int kb, int row0) {
        auto one = [&](uint32_t dst, int c0, int c2) {
          asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                       ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(row0), "r"(c2) : "memory");
        };
        if (h.flat) {
#pragma unroll
          for (int j = 0; j < IS_KPS; ++j) one(to + j * box, (kb + j) * IG_BK, 0);
        } else one(to, 0, kb);
      };
      const uint32_t xat = IS_KPS * IG_WBOX;
      const int first = min(ns, h.stages);
      int kb = s0 * IS_KPS;
      if (!p.w_ready) ig_wait_grid();
      for (int i = 0; i < first; ++i) {
        ig_expect(full0 + i * 8, STAGE);
        load(ring0 + i * STAGE, full0 + i * 8, &wmap, IG_WBOX, kb + i * IS_KPS, n0);
      }
      if (p.w_ready) ig_wait_grid();
      ig_next_grid();
      for (int i = 0; i < first; ++i, kb += IS_KPS) load(ring0 + i * STAGE + xat, full0 + i * 8, &xmap, XBOX, kb, m0);
      uint32_t at = ring0, bar = full0, ph = 0;
      for (int i = first; i < ns; ++i, kb += IS_KPS) {
        ig_wait(bar + EMPTY, ph, p.status, 41, abortw);
        ig_expect(bar, STAGE);
        load(at, bar, &wmap, IG_WBOX, kb, n0);
        load(at + xat, bar, &xmap, XBOX, kb, m0);
        at += STAGE; bar += 8;
        if (at == ring_end) { at = ring0; bar = full0; ph ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // One thread, and as few instructions a stage as can be: with few tokens an MMA is short and this loop is what a CTA
    // without a split is bound by (170 ns a k-block when the whole warp walked it and elected a lane every time, 92 so).
    if (ig_elect()) {
      constexpr uint32_t IDESC = ig_idesc(IG_BN, NT);
      const uint64_t a0 = ig_desc(ring0), b0 = ig_desc(ring0 + IS_KPS * IG_WBOX);
      uint64_t ad = a0, bd = b0;
      uint32_t at = ring0, bar = full0, ph = 0;
      ig_wait_grid();                                     // (no tile is complete before, and the bounded waits start counting here)
      for (int i = 0; i < ns; ++i) {
        ig_wait(bar, ph, p.status, 42, abortw);
        ig_fence_after();
#pragma unroll
        for (int j = 0; j < IS_KPS; ++j) ig_mma_stage<1>(tmem, ad + j * (IG_WBOX >> 4), bd + j * (XBOX >> 4), IDESC, i == 0 && j == 0);
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(i + 1 < ns ? bar + EMPTY : smem_u32(&acc_full)) : "memory");
        at += STAGE; bar += 8; ad += STAGE >> 4; bd += STAGE >> 4;
        if (at == ring_end) { at = ring0; bar = full0; ad = a0; bd = b0; ph ^= 1; }
      }
    }
    __syncwarp();
  } else {
    ig_wait_grid();
    for (int t = tid - 64; t < mt; t += 128) s_sx[t] = p.x_scale[m0 + t];
    if (mine) {
      sw = p.w_scale[n];
      if (p.bias != nullptr) bias = El<T>::ld((const T*)p.bias + n);
      if (p.res != nullptr) {
        const T* res = (const T*)p.res + (long long)(m0 + t0) * p.res_rs + n;
#pragma unroll 8
        for (int t = 0; t < nt; ++t) s_res[t * IG_BN + row] = res[t * p.res_rs];
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");        // s_sx is written
    ig_wait_warp(smem_u32(&acc_full), 0, p.status, 43, abortw);    // (the last stage's MMAs: all before them are done too)
    ig_fence_after();
  }
  const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
  T* y = (T*)p.y + (long long)(m0 + t0) * p.y_rs + n;
  auto finish = [&](int t, const int (&acc)[8]) {          // tokens t .. t + 7 of this CTA's
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = p.res != nullptr && t + i < nt ? El<T>::ld(s_res + (t + i) * IG_BN + row) : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (t + i < nt) El<T>::st(y + (t + i) * p.y_rs, (float)acc[i] * sw * s_sx[t0 + t + i] + bias + r[i]);
  };
  if (S == 1) {
    if (warp >= 2) {
      for (int t = 0; t < nt; t += 8) {
        int v[8];
        ig_ld8(lanes + (uint32_t)t, v);
        if (mine) finish(t, v);
      }
    }
  } else {
    ig_cluster_wait();
    if (warp >= 2) {
      for (int o = 0; o * h.per < mt; ++o) {               // tokens o * per ... to the CTA that finishes them
        const uint32_t to = ig_mapa(smem_u32(xch + rank * h.per * IG_BN + row), o);
        for (int t = 0; t < h.per && o * h.per + t < mt; t += 8) {
          int v[8];
          ig_ld8(lanes + (uint32_t)(o * h.per + t), v);
#pragma unroll
          for (int i = 0; i < 8; ++i) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + (t + i) * (IG_BN * 4)), "r"(v[i]) : "memory");
        }
      }
    }
    ig_cluster_arrive();
    ig_cluster_wait();
    if (mine) {
      for (int t = 0; t < nt; t += 8) {
        int v[8] = {};
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += xch[(s * h.per + t + i) * IG_BN + row];
        finish(t, v);
      }
    }
  }
  ig_fence_before();
  __syncthreads();
  ig_settle(abortw);
  if (warp == 1) {
    ig_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
  }
}

// ---- many tokens: pairs of SMs ------------------------------------------------------------------------
// A pair of CTAs works on 256 channels x NT tokens with one MMA (cta_group::2, M = 256): each holds its 128 channels and
// half of the tokens, so a stage costs 128 + NT / 2 rows of loads for 128 x NT products a byte of K -- two thirds of what
// one CTA alone would load for its 128 x NT, which is what the L2 cannot feed (it gives some 13 TB/s).  8192 x 8192 -> 8192
// with a residual 330 - 365 us (3.3 - 3.0 POP/s, as the power cap lets it); 16384 x 4096 -> 6177 276 us; the tensor pipe is 84 to 87 % active.  The pairs walk over the tiles
// (persistent); the accumulator is double-buffered in TMEM, so a tile's epilogue runs under the next tile's MMAs.
// Warp 0 = TMA producer (its copies complete on the pair's first CTA's barrier), warp 1 = MMA issuer (first CTA only) and
// TMEM owner, warps 2-9 = epilogue, two warps per 32 channels with half of the tokens each.
constexpr int IP_EPI = 8, IP_THREADS = 64 + 32 * IP_EPI;
constexpr long long IP_GROUP_BYTES = 40 << 20;           // weights that are walked together: what stays in L2
constexpr int ip_kps(int nt) { return nt == 256 ? 1 : 2; }  // k-blocks per stage
constexpr int ip_stages(int nt) { return nt == 256 ? 6 : nt == 128 ? 4 : 5; }
constexpr int ip_smem(int nt) { return 1024 + ip_stages(nt) * ip_kps(nt) * (IG_WBOX + nt / 2 * IG_BK) + (2 * ip_stages(nt) + 4) * 8 + 16; }
static_assert(ip_smem(64) + 2 * 64 * 4 + 64 <= IG_MAX_SMEM && ip_smem(128) + 2 * 128 * 4 + 64 <= IG_MAX_SMEM &&
              ip_smem(256) + 2 * 256 * 4 + 64 <= IG_MAX_SMEM, "ring does not fit in shared memory");

__device__ __forceinline__ void ip_tile(const Int8GemmParams& p, int id, int& ct, int& tt) {
  const int span = p.group * p.ttiles, g = id / span, left = min(p.group, p.ctiles - g * p.group), r = id - g * span;
  ct = g * p.group + r % left;
  tt = r / left;
}
__device__ __forceinline__ void ip_commit(uint32_t bar) {   // arrives at the barrier of that offset in both CTAs
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((uint16_t)3) : "memory");
}

template <typename T, int NT>
__global__ void __launch_bounds__(IP_THREADS, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, Int8GemmParams p) {
  constexpr int KPS = ip_kps(NT), STAGES = ip_stages(NT), XBOX = NT / 2 * IG_BK, STAGE = KPS * (IG_WBOX + XBOX);
  constexpr uint32_t EMPTY = STAGES * 8;
  constexpr uint32_t COLS = 2 * NT;
  extern __shared__ unsigned char ip_raw[];
  unsigned char* smem = ip_raw + ((1024u - (smem_u32(ip_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);     // first CTA's: both CTAs' copies of a stage
  uint64_t* empty = full + STAGES;                                        // each CTA's own
  uint64_t* acc_full = empty + STAGES;                                    // [2] each CTA's own
  uint64_t* acc_empty = acc_full + 2;                                     // [2] first CTA's: all epilogue warps of the pair
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  __shared__ float s_sx[2][NT];
  __shared__ int s_abort;
  int* const abortw = &s_abort;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = p.ctiles * p.ttiles;
  const uint32_t ring0 = smem_u32(smem), ring_end = ring0 + STAGES * STAGE, full0 = smem_u32(full);
  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < STAGES; ++i) { tma::mbar_init(&full[i], 1); tma::mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { tma::mbar_init(&acc_full[i], 1); tma::mbar_init(&acc_empty[i], 2 * IP_EPI); }
    tma::fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    ig_fence_before();
  }
  __syncthreads();
  ig_cluster_arrive();
  ig_cluster_wait();                                                      // both CTAs' barriers are ready
  ig_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (ig_elect()) {
      const bool flat = p.K % IG_BK != 0;
      const uint32_t to_lead = ig_mapa(full0, 0) - full0;    // this CTA's shared memory -> the first CTA's
      uint32_t at = ring0, bar = full0, ph = 1;              // (the first round finds every stage free)
      // k-blocks kb ... of `map` from row `row`, to `to`
      auto load = [&](uint32_t to, uint32_t arrive, const CUtensorMap* map, int box, int kb, int row) {
        auto one = [&](uint32_t dst, int c0, int c2) {
          asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];"
                       ::"r"(dst), "l"(map), "r"(arrive + to_lead), "r"(c0), "r"(row), "r"(c2) : "memory");
        };
        if (flat) {
#pragma unroll
          for (int j = 0; j < KPS; ++j) one(to + j * box, (kb + j) * IG_BK, 0);
        } else one(to, 0, kb);
      };
      int ct, tt, early = 0;                                 // stages of the first tile whose weights are requested ahead
      if (p.w_ready && pair < tiles) {
        ip_tile(p, pair, ct, tt);
        early = min((p.nkb + KPS - 1) / KPS, STAGES);
        for (int i = 0; i < early; ++i) {
          if (rank == 0) ig_expect(full0 + i * 8, 2 * STAGE);
          load(ring0 + i * STAGE, full0 + i * 8, &wmap, IG_WBOX, i * KPS, ct * 2 * IG_BN + rank * IG_BN);
        }
      }
      ig_wait_grid();
      ig_next_grid();
      for (int id = pair; id < tiles; id += pairs) {
        ip_tile(p, id, ct, tt);
        const int n0 = ct * 2 * IG_BN + rank * IG_BN, m0 = tt * NT + rank * (NT / 2);
        for (int kb = 0; kb < p.nkb; kb += KPS) {            // (what lies behind K is zero)
          if (early > 0) --early;
          else {
            ig_wait(bar + EMPTY, ph, p.status, 44, abortw);
            if (rank == 0) ig_expect(bar, 2 * STAGE);
            load(at, bar, &wmap, IG_WBOX, kb, n0);
          }
          load(at + KPS * IG_WBOX, bar, &xmap, XBOX, kb, m0);
          at += STAGE; bar += 8;
          if (at == ring_end) { at = ring0; bar = full0; ph ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && ig_elect()) {
      constexpr uint32_t IDESC = ig_idesc(2 * IG_BN, NT);
      const uint64_t a0 = ig_desc(ring0), b0 = ig_desc(ring0 + KPS * IG_WBOX);
      uint64_t ad = a0, bd = b0;
      uint32_t at = ring0, bar = full0, ph = 0;
      int j = 0;
      ig_wait_grid();                                       // (the bounded waits start counting here)
      for (int id = pair; id < tiles; id += pairs, ++j) {
        if (j >= 2) { ig_wait(smem_u32(&acc_empty[j & 1]), (j / 2 - 1) & 1, p.status, 45, abortw); ig_fence_after(); }
        const uint32_t dcol = tmem + (uint32_t)((j & 1) * NT);
        for (int kb = 0; kb < p.nkb; kb += KPS) {
          ig_wait(bar, ph, p.status, 46, abortw);
          ig_fence_after();
#pragma unroll
          for (int q = 0; q < KPS; ++q) ig_mma_stage<2>(dcol, ad + q * (IG_WBOX >> 4), bd + q * (XBOX >> 4), IDESC, kb == 0 && q == 0);
          ip_commit(bar + EMPTY);
          at += STAGE; bar += 8; ad += STAGE >> 4; bd += STAGE >> 4;
          if (at == ring_end) { at = ring0; bar = full0; ad = a0; bd = b0; ph ^= 1; }
        }
        ip_commit(smem_u32(&acc_full[j & 1]));
      }
    }
    __syncwarp();
  } else {
    ig_wait_grid();
    const int et = tid - 64, quarter = warp & 3, half = (warp - 2) >> 2, row = quarter * 32 + lane;
    int j = 0;
    for (int id = pair; id < tiles; id += pairs, ++j) {
      int ct, tt;
      ip_tile(p, id, ct, tt);
      const int n = ct * 2 * IG_BN + rank * IG_BN + row, m0 = tt * NT, b = j & 1;
      const bool mine = n < p.N;
      const int mt = min(NT, p.M - m0);
      for (int t = et; t < NT; t += 32 * IP_EPI) s_sx[b][t] = t < mt ? p.x_scale[m0 + t] : 0.f;
      const float sw = mine ? p.w_scale[n] : 0.f;
      const float bias = mine && p.bias != nullptr ? El<T>::ld((const T*)p.bias + n) : 0.f;
      asm volatile("bar.sync 1, %0;" ::"n"(32 * IP_EPI) : "memory");
      ig_wait_warp(smem_u32(&acc_full[b]), (j >> 1) & 1, p.status, 47, abortw);
      ig_fence_after();
      for (int c = half * (NT / 2); c < (half + 1) * (NT / 2); c += 32) {
        uint32_t v[32];
        ig_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * NT + c), v);
        if (mine && c < mt) {
          T* y = (T*)p.y + (long long)(m0 + c) * p.y_rs + n;
          float r[32];
          if (p.res != nullptr) {                          // rows past M read the last one again: no branch around the loads
            const T* res = (const T*)p.res + (long long)(m0 + c) * p.res_rs + n;
#pragma unroll
            for (int t = 0; t < 32; ++t) { r[t] = El<T>::ld(res); res += c + t + 1 < mt ? p.res_rs : 0; }
          }
#pragma unroll
          for (int t = 0; t < 32; ++t, y += p.y_rs) {
            const float v1 = (float)(int)v[t] * sw * s_sx[b][c + t] + bias;
            if (c + t < mt) El<T>::st(y, p.res != nullptr ? v1 + r[t] : v1);
          }
        }
      }
      ig_fence_before();
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(ig_mapa(smem_u32(&acc_empty[b]), 0)) : "memory");
    }
  }
  ig_fence_before();
  __syncthreads();
  ig_settle(abortw);
  ig_cluster_arrive();                                   // neither CTA leaves while the other may still reach its memory
  ig_cluster_wait();
  if (warp == 1) {
    ig_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
  }
}

// Self-test of these waits, on barriers that nobody arrives at: warp 0 gives up after `poll_limit` polls, warp 1, with the
// full limit, as soon as it sees the abort word; then every thread passes ig_settle.
__global__ void ig_selftest_kernel(int poll_limit, int* status, int* report) {
  __shared__ uint64_t bars[2];
  __shared__ int s_abort;
  if (threadIdx.x == 0) {
    s_abort = 0;
    tma::mbar_init(&bars[0], 1);
    tma::mbar_init(&bars[1], 1);
    tma::fence_barrier_init();
  }
  __syncthreads();
  const int who = threadIdx.x / 32;
  const long long t0 = clock64();
  if (who == 0) {
    if (ig_elect()) ig_wait(smem_u32(&bars[0]), 0, status, 48, &s_abort, poll_limit);
    __syncwarp();
  } else ig_wait_warp(smem_u32(&bars[1]), 0, status, 49, &s_abort);
  const long long dt = clock64() - t0;
  if (threadIdx.x % 32 == 0) {
    report[2 * who] = (int)ig_try(smem_u32(&bars[who]), 0);
    report[2 * who + 1] = dt > 0x7fffffffLL ? 0x7fffffff : (int)dt;
  }
  __syncthreads();
  ig_settle(&s_abort);
  if (threadIdx.x == 0) report[4] = s_abort;
}

// ---- launch ----------------------------------------------------------------------------------------------
struct Int8Plan { bool pair; int nt, split, smem; };   // smem: bytes a CTA of the split kernel may use

template <typename T, typename K, typename... A>
int ig_launch(K kernel, int smem, dim3 grid, int threads, int cluster, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = grid; lc.blockDim = dim3(threads); lc.dynamicSmemBytes = smem; lc.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  lc.attrs = at; lc.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&lc, kernel, args...);
  if (e != cudaSuccess) { coda_set_error("int8_gemm: %s", cudaGetErrorString(e)); cudaGetLastError(); return CODA_ERR_LAUNCH; }
  return CODA_OK;
}

// Shared memory of a split launch: the ring takes what residual tile and exchange leave of `smem`.
template <typename T>
SplitShape split_shape(const Int8Plan& q, const Int8GemmParams& p) {
  SplitShape h = {};
  h.split = q.split; h.flat = p.K % IG_BK != 0;
  const int mt = p.M < q.nt ? p.M : q.nt;
  h.per = ((mt + q.split - 1) / q.split + 7) / 8 * 8;
  h.res = p.res != nullptr ? h.per * IG_BN * (int)sizeof(T) : 0;
  h.xch = q.split > 1 ? q.split * h.per * IG_BN * 4 : 0;
  const int stage = IS_KPS * (IG_BN + q.nt) * IG_BK, ns = ((p.nkb + IS_KPS - 1) / IS_KPS + q.split - 1) / q.split;
  const int fit = (q.smem - 1024 - h.res - h.xch) / stage;
  h.stages = fit < ns ? fit : ns;
  h.ring = h.stages * stage;
  h.total = 1024 + h.ring + h.res + h.xch;
  return h;
}

template <typename T, int NT>
int launch_split(const Int8Plan& q, const Int8GemmParams& p, const CUtensorMap& xm, const CUtensorMap& wm, cudaStream_t s) {
  static coda_device_once once;
  coda_on_first_use(once, [] {
    cudaFuncSetAttribute(int8_split_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, IS_SMEM_WHOLE);
  });
  const SplitShape h = split_shape<T>(q, p);
  CODA_REQUIRE(h.stages > 0, CODA_ERR_LIMIT, "int8_gemm: no room for a stage");
  return ig_launch<T>(int8_split_kernel<T, NT>, h.total, dim3(p.ctiles * q.split, p.ttiles), IS_THREADS, q.split, s, xm, wm, p, h);
}

// Groups of channel tiles, each over all tokens before the next: as even as they can be with the weights of one in L2.
// 8192 x 8192 -> 8192 (us): groups of 4 / 8 / 16 / 32 tiles 342 / 331 / 323 / 362; 16384 x 4096 -> 6177: of 8 / 16 / 25 288 / 281 / 275.
template <typename T, int NT>
int launch_pair(Int8GemmParams p, const CUtensorMap& xm, const CUtensorMap& wm, cudaStream_t s) {
  static coda_device_once once;
  const int sms = coda_on_first_use(once, [] {
    cudaFuncSetAttribute(int8_pair_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, ip_smem(NT));
  });
  const long long tiles = (long long)p.ctiles * p.ttiles, fit = IP_GROUP_BYTES / (2 * IG_BN * (long long)p.K);
  const long long groups = (p.ctiles + (fit > 1 ? fit : 1) - 1) / (fit > 1 ? fit : 1);
  p.group = (int)((p.ctiles + groups - 1) / groups);
  const int pairs = (int)(tiles < sms / 2 ? tiles : sms / 2);
  return ig_launch<T>(int8_pair_kernel<T, NT>, ip_smem(NT), dim3(2 * pairs), IP_THREADS, 2, s, xm, wm, p);
}

struct Int8Operands { const int8_t* x; long long x_rs; const int8_t* w; long long w_rs; };

template <typename T>
int launch_plan(const Int8Plan& q, const Int8Operands& o, Int8GemmParams p, cudaStream_t s) {
  const int rows = q.pair ? 2 * IG_BN : IG_BN;
  p.ctiles = (p.N + rows - 1) / rows;
  p.ttiles = (p.M + q.nt - 1) / q.nt;
  CUtensorMap xm, wm;
  const bool ok = q.pair ? tmaps::byte_map(&xm, o.x, p.M, p.K, o.x_rs, q.nt / 2, ip_kps(q.nt)) && tmaps::byte_map(&wm, o.w, p.N, p.K, o.w_rs, IG_BN, ip_kps(q.nt))
                         : tmaps::byte_map(&xm, o.x, p.M, p.K, o.x_rs, q.nt, IS_KPS) && tmaps::byte_map(&wm, o.w, p.N, p.K, o.w_rs, IG_BN, IS_KPS);
  CODA_REQUIRE(ok, CODA_ERR_LAUNCH, "int8_gemm: cuTensorMapEncodeTiled failed");
  if (q.pair) return q.nt == 64 ? launch_pair<T, 64>(p, xm, wm, s) : q.nt == 128 ? launch_pair<T, 128>(p, xm, wm, s) : launch_pair<T, 256>(p, xm, wm, s);
  return q.nt == 16 ? launch_split<T, 16>(q, p, xm, wm, s) : q.nt == 32 ? launch_split<T, 32>(q, p, xm, wm, s)
                                                            : launch_split<T, 64>(q, p, xm, wm, s);
}

// The plan that is estimated to be the quickest.  Microseconds beyond what every plan costs, fitted to every plan's time at
// 1008 sizes (M 1 .. 4096, K 128 .. 8192, N 200 .. 20000, bf16, back to back with cold weights): a k-block costs a CTA or pair
// so much, waves of tiles follow one another, and the bytes that go in and out, at a rate that was fitted with the rest (twice
// what HBM gives: loads and products overlap), add to that as the other leg of a right angle.
Int8Plan choose_plan(long long M, long long K, long long N) {
  auto up = [](long long a, long long b) { return (a + b - 1) / b; };
  const long long nkb = up(K, IG_BK);
  const double bytes = (double)(N * K + M * K + 2 * M * N) / 13.3e6;
  Int8Plan best = {};
  double least = 1e30;
  for (int i = 0; i < 3; ++i) {                            // pairs of SMs, 74 of them
    static const double block[3] = {0.163, 0.185, 0.279}, tail[3] = {1.06, 1.23, 1.45};
    const int nt = 64 << i;
    const double run = (double)up(up(N, 2 * IG_BN) * up(M, nt), 74) * fmax((double)up(nkb, ip_kps(nt)) * ip_kps(nt) * block[i], tail[i]);
    const double t = sqrt(run * run + bytes * bytes) + tail[i];
    if (t < least) { least = t; best = Int8Plan{true, nt, 1, 0}; }
  }
  if (M > 512) return best;
  const int i = M <= 16 ? 0 : M <= 32 ? 1 : 2, nt = 16 << i;
  for (int split = 1, at = 0; split <= 8 && split <= up(nkb, IS_KPS); split *= 2, ++at) {   // clusters that share a tile's K
    static const double block[3] = {0.101, 0.105, 0.283}, tail1[3] = {0.37, 1.09, 2.53}, tail[3] = {1.43, 1.93, 2.27};
    static const int resident[4] = {148, 148, 132, 120};   // CTAs that run at once in clusters of 1, 2, 4, 8
    const long long ctas = up(N, IG_BN) * up(M, nt) * split;
    const bool half = nt < 64 && ctas > resident[at];      // two CTAs to an SM: the ring in half of its shared memory
    if (split == 8 && half) break;
    const double waves = (double)up(ctas, resident[at] * (half ? 2 : 1));
    const double run = waves * (double)(up(up(nkb, IS_KPS), split) * IS_KPS) * block[i] * (half && ctas > 148 ? 3.1 : 1.0);
    const double t = sqrt(run * run + bytes * bytes) + 1.47 * (waves - 1) + (split == 1 ? tail1[i] : tail[i]);
    if (t < least) { least = t; best = Int8Plan{false, nt, split, half ? IS_SMEM_HALF : IS_SMEM_WHOLE}; }
  }
  return best;
}

}  // namespace

extern "C" int coda_b200_int8_gemm(int32_t dtype, int32_t M, int32_t K, int32_t N, const int8_t* x, int64_t x_rs, const float* x_scale,
                                   const int8_t* w, int64_t w_rs, const float* w_scale, const void* bias,
                                   const void* residual, int64_t res_rs, void* y, int64_t y_rs, int32_t w_ready, int32_t* status, coda_stream_t stream) {
  CODA_REQUIRE((dtype == CODA_F32 || dtype == CODA_BF16) && M >= 0 && N > 0 && K > 0, CODA_ERR_ARG, "int8_gemm: dtype or sizes invalid");
  CODA_REQUIRE(K <= 131071, CODA_ERR_LIMIT, "int8_gemm: K = %d, the 32-bit sum holds at most 131071 products", K);
  CODA_REQUIRE(M <= 2147483000 && N <= 2147483000, CODA_ERR_LIMIT, "int8_gemm: M or N over 2147483000");
  if (M == 0) return CODA_OK;
  CODA_REQUIRE(x && x_scale && w && w_scale && y, CODA_ERR_ARG, "int8_gemm: null pointer");
  CODA_REQUIRE(((uintptr_t)x | (uintptr_t)w) % 16 == 0 && x_rs % 16 == 0 && w_rs % 16 == 0, CODA_ERR_ARG,
               "int8_gemm: rows of x and w must start on 16-byte boundaries");
  CODA_REQUIRE(((uintptr_t)y | (uintptr_t)bias | (uintptr_t)residual) % (dtype == CODA_F32 ? 4 : 2) == 0 &&
               ((uintptr_t)x_scale | (uintptr_t)w_scale | (uintptr_t)status) % 4 == 0, CODA_ERR_ARG,
               "int8_gemm: tensors must start on a boundary of their elements");
  CODA_REQUIRE(x_rs >= K && w_rs >= K && y_rs >= N && (residual == nullptr || res_rs >= N), CODA_ERR_ARG,
               "int8_gemm: row strides shorter than a row");
  Int8GemmParams p = {};
  p.M = M; p.N = N; p.K = K; p.nkb = (K + IG_BK - 1) / IG_BK;
  p.x_scale = x_scale; p.w_scale = w_scale; p.bias = bias; p.res = residual; p.res_rs = res_rs; p.y = y; p.y_rs = y_rs; p.status = status; p.w_ready = w_ready;
  const Int8Operands o{x, x_rs, w, w_rs};
  if (dtype == CODA_F32) return launch_plan<float>(choose_plan(M, K, N), o, p, (cudaStream_t)stream);
  return launch_plan<bf16>(choose_plan(M, K, N), o, p, (cudaStream_t)stream);
}

extern "C" int coda_b200_selftest_int8_wait(int32_t poll_limit, int32_t* status, int32_t* report, coda_stream_t stream) {
  CODA_REQUIRE(status && report, CODA_ERR_ARG, "selftest_int8_wait: null pointer");
  CODA_REQUIRE(poll_limit > 0 && poll_limit <= (1 << 16), CODA_ERR_ARG, "selftest_int8_wait: poll_limit must be in 1..65536");
  ig_selftest_kernel<<<1, 64, 0, (cudaStream_t)stream>>>(poll_limit, status, report);
  CODA_CHECK_LAUNCH("selftest_int8_wait");
  return CODA_OK;
}
