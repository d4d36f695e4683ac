// Rows around the 8-bit projections: RMS norm with the residual's addition, rows to 8 bits, and back.
//
//   s = x + residual                        (written in the type of x: the residual stream)
//   y = s * rsqrt(mean(s^2) + eps) * weight (of the unrounded s)
//   out = y rounded to the type of x, or in 8 bits:  a = max|y|,  scale = a / 127,  q = rint(127 y / a), ties to even
//
// Everything between the loads and the stores is fp32, each output is rounded once.  A row whose largest magnitude is
// under 2^-100 becomes zeros with scale 0 (127 / a would leave fp32's range); a row that holds a NaN or an infinity
// becomes zeros with scale NaN, so that whatever is computed from it is NaN.
// Bound: HBM (x, residual, s, one byte of q an element), and for the rows of a decode step the latency of one load,
// two reductions and one store.  So a row stays in the registers of the threads that loaded it: one pass over memory.
// 16384 x 4096 bf16: norm with residual to 8 bits 69 us = 6.8 TB/s (1.04 of the measured copy), rows to 8 bits 33 us = 6.1, back
// 34 us = 5.8; 32 x 4096 under 2 us each.  Rows that are no whole vectors: 57 us for the norm of 8192 x 4094 bf16 (36 where
// they are), 72 us for 8192 x 4095 (120 before odd rows were read by aligned words).
#include "coda_common.cuh"
#include <type_traits>

namespace {

// The next kernel on the stream may come as soon as this one's CTAs are there -- a product then has its barriers, tensor
// memory and, where its weights are old (w_ready), a first ring of them before these rows are done -- and every access of
// this kernel's own waits for the one before it.
__device__ __forceinline__ void rows_chain() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

struct RowsParams {
  long long rows;
  int dim;
  const void* x; long long x_rs;
  const void* res; long long res_rs;     // or null
  const void* w;                         // norm weight, null: rows are quantised as they are
  float eps;
  void* sum; long long sum_rs;           // or null
  void* y; long long y_rs;               // normed rows in the type of x, or null
  int8_t* q; long long q_rs;             // 8-bit rows, or null
  float* scale;
};

// EPC elements in one access (16, 4, 2 bytes ...; the caller has checked the alignment), as they lie in memory ...
template <typename T, int EPC> struct Chunk {
  static constexpr int BYTES = EPC * (int)sizeof(T), WORDS = (BYTES + 3) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (BYTES == 16) { const uint4 u = *reinterpret_cast<const uint4*>(p); w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; }
    else if constexpr (BYTES == 4) w[0] = *reinterpret_cast<const uint32_t*>(p);
    else w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
  // ... and in fp32
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float(i % 2 == 0 ? w[i / 2] << 16 : w[i / 2] & 0xffff0000u);
  }
};
template <typename T, int EPC> __device__ __forceinline__ void st_chunk(T* p, const float (&v)[EPC]) {
  if constexpr (EPC == 1) El<T>::st(p, v[0]);
  else {
    uint32_t w[EPC * sizeof(T) / 4];
#pragma unroll
    for (int i = 0; i < (int)(EPC * sizeof(T) / 4); ++i) {
      if constexpr (sizeof(T) == 2) { __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]); w[i] = *reinterpret_cast<uint32_t*>(&b); }
      else w[i] = __float_as_uint(v[i]);
    }
    if constexpr (EPC * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}
// What 8-bit row a largest magnitude (its bits: NaN and infinity are the largest) makes: scale, and the factor to 127.
// (inv is 0 where the row becomes zeros)
struct Q8 { float a, scale, inv; };
__device__ __forceinline__ Q8 row_scale(uint32_t amax) {
  const float a = __uint_as_float(amax);
  if (amax >= 0x7f800000u) return Q8{0.f, __uint_as_float(0x7fc00000u), 0.f};
  if (a < 7.888609e-31f) return Q8{0.f, 0.f, 0.f};
  return Q8{a, __fdiv_rn(a, 127.f), __fdiv_rn(127.f, a)};
}
// q = rint(127 y / a), ties to even.  To round, 1.5 * 2^23 is added: its last bit is worth 1, and the low byte of the sum's
// bits is q.  y * inv is within 127 * 2^-24 of the quotient, so its nearest integer is right unless it lies that close to a
// half.  Half of a row's largest value is such a tie, 63.5: without more, 1 of some 6000 values of random bf16 rows
// came out a step off (and 1 of 20000 by a division by the scale: two roundings miss ties too).  How far that is looked at:
// Q8_SHORT  bf16 rows as they are: a quotient of two 8-bit values is a half or 2 / (512 * 255) away from one at the least (254 y -
//           256 a is even; further above one half), so y * inv is rounded to multiples of 2^-15 first: that restores the
//           halves and makes none.
// Q8_LONG   float32 rows as they are: near a half 127 y is compared with the half's multiple of a, in products split into two
//           floats each, by a call: 1 of 50000 random values is that near (8192 x 4096: 26.9 us, 25.9 without; 28.7 with the
//           comparison for every value).
// Q8_PLAIN  normed rows, whose y has roundings of its own that weigh more.
enum { Q8_SHORT, Q8_LONG, Q8_PLAIN };
constexpr float Q8_MAGIC = 12582912.f, Q8_SNAP = 384.f, Q8_NEAR = 0.49999f;
__device__ __noinline__ float q8_near_half(float y, float q, float d, float a) {   // y * inv = q + d
  const float k = a > 1.f ? 0.00390625f : 1.f, c = 127.f * k;                     // (127 y of rows near the end of the range)
  a *= k;
  const float h = q + copysignf(0.5f, d), p = y * c, s = h * a;
  const float over = (p - s) + (fmaf(y, c, -p) - fmaf(h, a, -s));                 // 127 y - h a: p - s is exact, both rests are
  return over > 0.f ? h + 0.5f : over < 0.f ? h - 0.5f : rintf(h);
}
// Elements of a row that hold y to 8 bits, in the low bytes of w[i].
template <int EPC, int KIND> __device__ __forceinline__ void to_q8(const float (&v)[EPC], const Q8& r, uint32_t (&w)[EPC]) {
  if (r.inv == 0.f) {                                                              // (0 * infinity would be no zero)
#pragma unroll
    for (int i = 0; i < EPC; ++i) w[i] = 0u;
    return;
  }
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < EPC; ++i) {
    if constexpr (KIND == Q8_SHORT) w[i] = __float_as_uint(fmaf(v[i], r.inv, Q8_SNAP) + (Q8_MAGIC - Q8_SNAP));
    else {
      const float g = fmaf(v[i], r.inv, Q8_MAGIC);
      if constexpr (KIND == Q8_LONG) far = fmaxf(far, fabsf(fmaf(v[i], r.inv, Q8_MAGIC - g)));
      w[i] = __float_as_uint(g);
    }
  }
  if (KIND == Q8_LONG && far > Q8_NEAR) {
#pragma unroll
    for (int i = 0; i < EPC; ++i) {
      const float q = __uint_as_float(w[i]) - Q8_MAGIC, d = fmaf(v[i], r.inv, -q);
      if (fabsf(d) > Q8_NEAR) w[i] = __float_as_uint(q8_near_half(v[i], q, d, r.a) + Q8_MAGIC);
    }
  }
}
template <int EPC, int KIND> __device__ __forceinline__ void st_q(int8_t* p, const float (&v)[EPC], const Q8& r) {
  uint32_t b[EPC];
  to_q8<EPC, KIND>(v, r, b);
  if constexpr (EPC == 1) *p = (int8_t)b[0];
  else if constexpr (EPC == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)__byte_perm(b[0], b[1], 0x40);
  else {
    uint32_t w[EPC / 4];
#pragma unroll
    for (int i = 0; i < EPC / 4; ++i)
      w[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x40), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x40), 0x5410);
    if constexpr (EPC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// A chunk of a row of `dim` elements from element `at`; elements outside the row are zeros and are not stored.  STAGGER: chunks
// are the aligned words of a bf16 row that may start between two (at is -1, 1, 3 ... then): the first and the last word may
// hold one element of this row only, and what lies in the other half is neither read nor written.
template <typename T, int EPC, bool STAGGER>
__device__ __forceinline__ void ld_part(Chunk<T, EPC>& c, const T* row, int at, int dim) {
  if (at >= 0 && at + (STAGGER ? 1 : 0) < dim) { c.load(row + at); return; }
#pragma unroll
  for (int i = 0; i < Chunk<T, EPC>::WORDS; ++i) c.w[i] = 0u;
  if constexpr (STAGGER) {
    if (at < 0) c.w[0] = (uint32_t)*reinterpret_cast<const uint16_t*>(row) << 16;
    else if (at < dim) c.w[0] = *reinterpret_cast<const uint16_t*>(row + at);
  }
}
template <typename T, int EPC, bool STAGGER>
__device__ __forceinline__ void st_part(T* row, int at, int dim, const float (&v)[EPC]) {
  if (at >= 0 && at + (STAGGER ? 1 : 0) < dim) { st_chunk<T, EPC>(row + at, v); return; }
  if constexpr (STAGGER) {
    if (at < 0) El<T>::st(row, v[1]);
    else if (at < dim) El<T>::st(row + at, v[0]);
  }
}
// Sum / maximum over the threads of a row: a warp (CTA of several rows) or the whole CTA (one row).
template <bool CTA> __device__ __forceinline__ float row_sum(float v, float* sh) {
  v = warp_sum(v);
  if constexpr (CTA) {
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    const int n = blockDim.x >> 5;
    v = warp_sum((int)(threadIdx.x & 31) < n ? sh[threadIdx.x & 31] : 0.f);
  }
  return v;
}
template <bool CTA> __device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* sh) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (CTA) {
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    const int n = blockDim.x >> 5;
    v = __reduce_max_sync(0xffffffffu, (int)(threadIdx.x & 31) < n ? sh[threadIdx.x & 31] : 0u);
  }
  return v;
}

// The row in registers: thread t of the row's TPR threads holds chunks t, t + TPR, ... (NCH of them, EPC elements each).
// All its loads (x, residual, weight) are out before the first is used.
template <typename T, int EPC, int NCH, int THREADS, bool CTA, bool NORM, bool STAGGER>
__global__ void __launch_bounds__(THREADS) int8_rows_kernel(RowsParams p) {
  __shared__ float sh_sum[32];
  __shared__ uint32_t sh_max[32];
  const int tpr = CTA ? blockDim.x : 32;
  const int t = CTA ? threadIdx.x : threadIdx.x & 31;
  const long long row = CTA ? (long long)blockIdx.x : (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  rows_chain();
  if (!CTA && row >= p.rows) return;
  const T* x = (const T*)p.x + row * p.x_rs;
  const bool res = NORM && p.res != nullptr;
  const int shift = STAGGER ? (int)((reinterpret_cast<uintptr_t>(x) >> 1) & 1) : 0;
  auto first = [&](int j) { return (t + j * tpr) * EPC - shift; };           // first element of chunk j
  float v[NCH][EPC];
  Chunk<T, EPC> cw[NORM ? NCH : 1];
  {
    Chunk<T, EPC> cx[NCH], cr[NORM ? NCH : 1];
#pragma unroll
    for (int j = 0; j < NCH; ++j) ld_part<T, EPC, STAGGER>(cx[j], x, first(j), p.dim);
    if (res) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) ld_part<T, EPC, STAGGER>(cr[j], (const T*)p.res + row * p.res_rs, first(j), p.dim);
    }
    if constexpr (NORM) {
      const T* w = (const T*)p.w;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        if constexpr (STAGGER) {                                              // (the weight's words do not move with the row's)
          const int at = first(j);
          cw[j].w[0] = (at >= 0 && at < p.dim ? (uint32_t)*reinterpret_cast<const uint16_t*>(w + at) : 0u) |
                       (at + 1 < p.dim ? (uint32_t)*reinterpret_cast<const uint16_t*>(w + at + 1) << 16 : 0u);
        } else ld_part<T, EPC, false>(cw[j], w, first(j), p.dim);
      }
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < EPC; ++i) v[j][i] = cx[j].get(i);
    if (res) {
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
#pragma unroll
        for (int i = 0; i < EPC; ++i) v[j][i] += cr[j].get(i);
        st_part<T, EPC, STAGGER>((T*)p.sum + row * p.sum_rs, first(j), p.dim, v[j]);
      }
    }
  }
  if constexpr (NORM) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < EPC; ++i) ss = fmaf(v[j][i], v[j][i], ss);
    const float inv = rsqrtf(__fdiv_rn(row_sum<CTA>(ss, sh_sum), (float)p.dim) + p.eps);
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < EPC; ++i) v[j][i] = v[j][i] * inv * cw[j].get(i);
  }
  if (NORM && p.q == nullptr) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) st_part<T, EPC, STAGGER>((T*)p.y + row * p.y_rs, first(j), p.dim, v[j]);
    return;
  }
  uint32_t amax = 0;                       // (elements outside the row are zeros)
#pragma unroll
  for (int j = 0; j < NCH; ++j)
#pragma unroll
    for (int i = 0; i < EPC; ++i) amax = max(amax, __float_as_uint(v[j][i]) & 0x7fffffffu);
  const Q8 to = row_scale(row_max<CTA>(amax, sh_max));
  int8_t* q = p.q + row * p.q_rs;
  constexpr int KIND = NORM ? Q8_PLAIN : sizeof(T) == 2 ? Q8_SHORT : Q8_LONG;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int at = first(j);
    if constexpr (STAGGER) {
      uint32_t b[EPC];
      to_q8<EPC, KIND>(v[j], to, b);
      if (at >= 0 && at < p.dim) q[at] = (int8_t)b[0];
      if (at + 1 < p.dim) q[at + 1] = (int8_t)b[1];
    } else if (at < p.dim) st_q<EPC, KIND>(q + at, v[j], to);
  }
  if (t == 0) p.scale[row] = to.scale;
}

// Rows longer than the registers of a CTA hold: the same in three passes, re-read from L2 where they fit it.
template <typename T>
__global__ void __launch_bounds__(1024) int8_rows_long_kernel(RowsParams p) {
  __shared__ float sh_sum[32];
  __shared__ uint32_t sh_max[32];
  rows_chain();
  const long long row = blockIdx.x;
  const T* x = (const T*)p.x + row * p.x_rs;
  const T* r = p.res != nullptr ? (const T*)p.res + row * p.res_rs : nullptr;
  const T* w = (const T*)p.w;
  auto at = [&](int d) { return r != nullptr ? El<T>::ld(x + d) + El<T>::ld(r + d) : El<T>::ld(x + d); };
  float inv = 1.f;
  if (w != nullptr) {
    float ss = 0.f;
    for (int d = threadIdx.x; d < p.dim; d += blockDim.x) { const float s = at(d); ss = fmaf(s, s, ss); }
    inv = rsqrtf(__fdiv_rn(row_sum<true>(ss, sh_sum), (float)p.dim) + p.eps);
  }
  auto normed = [&](float s, int d) { return w != nullptr ? s * inv * El<T>::ld(w + d) : s; };
  Q8 to{};
  if (p.q != nullptr) {
    uint32_t amax = 0;
    for (int d = threadIdx.x; d < p.dim; d += blockDim.x) amax = max(amax, __float_as_uint(normed(at(d), d)) & 0x7fffffffu);
    to = row_scale(row_max<true>(amax, sh_max));
    if (threadIdx.x == 0) p.scale[row] = to.scale;
  }
  for (int d = threadIdx.x; d < p.dim; d += blockDim.x) {
    const float s = at(d), y = normed(s, d);          // (sum may be x or residual itself: each element is read before it is written)
    if (p.q != nullptr) {
      const float one[1] = {y};
      if (w != nullptr) st_q<1, Q8_PLAIN>(p.q + row * p.q_rs + d, one, to);
      else st_q<1, sizeof(T) == 2 ? Q8_SHORT : Q8_LONG>(p.q + row * p.q_rs + d, one, to);
    }
    else El<T>::st((T*)p.y + row * p.y_rs + d, y);
    if (p.sum != nullptr) El<T>::st((T*)p.sum + row * p.sum_rs + d, s);
  }
}

// A warp per row where that is enough, else a CTA per row: few rows get a thread for every chunk (latency), many rows MANY
// chunks a thread (fewer warps to synchronise for the same bytes in flight; as many as fit in registers).
template <typename T, int EPC, bool NORM, bool STAGGER>
int launch_rows(const RowsParams& p, int sms, cudaStream_t s) {
  constexpr bool VEC = EPC * sizeof(T) == 16;
  constexpr int MANY = VEC ? 4 : NORM ? 8 : 16, WIDE = VEC && NORM ? 256 : 512;
  const long long chunks = ((long long)p.dim + (STAGGER ? 1 : 0) + EPC - 1) / EPC;
  const dim3 rows((unsigned)p.rows), warps((unsigned)((p.rows + 3) / 4));
  auto threads = [&](int nch) { return dim3((unsigned)((chunks + nch - 1) / nch + 31) / 32 * 32); };
  cudaError_t e;
  if (chunks <= 32) e = coda_launch_chained(int8_rows_kernel<T, EPC, 1, 128, false, NORM, STAGGER>, warps, dim3(128), 0, s, 1, p);
  else if (chunks <= 32 * MANY && p.rows > sms) e = coda_launch_chained(int8_rows_kernel<T, EPC, MANY, 128, false, NORM, STAGGER>, warps, dim3(128), 0, s, 1, p);
  else if (chunks <= 1024 && p.rows <= 2 * sms) e = coda_launch_chained(int8_rows_kernel<T, EPC, 1, 1024, true, NORM, STAGGER>, rows, threads(1), 0, s, 1, p);
  else if (chunks <= WIDE * MANY) e = coda_launch_chained(int8_rows_kernel<T, EPC, MANY, WIDE, true, NORM, STAGGER>, rows, threads(MANY), 0, s, 1, p);
  else if (chunks <= 1024 * MANY) e = coda_launch_chained(int8_rows_kernel<T, EPC, MANY, 1024, true, NORM, STAGGER>, rows, threads(MANY), 0, s, 1, p);
  else e = coda_launch_chained(int8_rows_long_kernel<T>, rows, dim3(1024), 0, s, 1, p);
  if (e != cudaSuccess) { coda_set_error("int8_rows: %s", cudaGetErrorString(e)); cudaGetLastError(); return CODA_ERR_LAUNCH; }
  return CODA_OK;
}

template <typename T>
int dispatch_rows(const RowsParams& p, cudaStream_t s) {
  static coda_device_once once;
  const int sms = coda_on_first_use(once, [] {});
  // whole chunks of `n` elements, every row of every tensor on a chunk's boundary (8-bit rows: n bytes)
  auto whole = [&](int n) {
    auto vec = [&](const void* q, long long rs, int bytes) { return q == nullptr || ((uintptr_t)q % bytes == 0 && rs % n == 0); };
    const int bytes = n * (int)sizeof(T);
    return p.dim % n == 0 && vec(p.x, p.x_rs, bytes) && vec(p.res, p.res_rs, bytes) && vec(p.w, 0, bytes) &&
           vec(p.sum, p.sum_rs, bytes) && vec(p.y, p.y_rs, bytes) && vec(p.q, p.q_rs, n);
  };
  auto go = [&](auto norm) {
    constexpr bool NORM = decltype(norm)::value;
    constexpr int V = 16 / (int)sizeof(T);
    if (whole(V)) return launch_rows<T, V, NORM, false>(p, sms, s);
    if constexpr (sizeof(T) == 2) {
      if (whole(2)) return launch_rows<T, 2, NORM, false>(p, sms, s);
      // all rows of the same number start alike: on a word, or between two
      auto alike = [&](const void* q, long long rs) { return q == nullptr || ((((uintptr_t)q ^ (uintptr_t)p.x) & 3) == 0 && ((rs ^ p.x_rs) & 1) == 0); };
      if ((uintptr_t)p.x % 2 == 0 && alike(p.res, p.res_rs) && alike(p.sum, p.sum_rs) && alike(p.y, p.y_rs)) return launch_rows<T, 2, NORM, true>(p, sms, s);
    }
    return launch_rows<T, 1, NORM, false>(p, sms, s);
  };
  return p.w != nullptr ? go(std::true_type{}) : go(std::false_type{});
}

// q * scale, rounded to T.  A thread takes the same E elements of DQ_ROWS rows, all of them requested before the first is used.
// WHOLE: E elements make 16 bytes of the output, rows of it start on such a boundary.  Else a warp's 256 elements of a row go
// through shared memory, so that its stores are neighbouring words all the same (8192 x 4095 bf16: 61 us an element a thread,
// 29 us so; 18 us is what whole rows of about that size take).  No pointer is __restrict__: the kernel ahead may still be writing q and
// scale when this one starts, and they must not pass for memory that is constant for its lifetime (loads ahead of the wait,
// or on the path that is not kept coherent).
template <typename T, int E, bool WHOLE, int DQ_ROWS>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(long long rows, int dim, const int8_t* q, long long q_rs,
                                                              const float* scale, T* out, long long out_rs,
                                                              int lanes) {
  __shared__ alignas(16) T seg[WHOLE ? 1 : 8][WHOLE ? 1 : 32 * E];
  const int local = threadIdx.x / lanes, per = blockDim.x / lanes, t = threadIdx.x - local * lanes;
  const long long row0 = (long long)blockIdx.x * per * DQ_ROWS + local;      // rows row0, row0 + per, ...
  rows_chain();
  if (local >= per) return;                                                  // (whole warps: lanes divides 256 or is a multiple of 32)
  const int n = (int)min((rows - row0 + per - 1) / per, (long long)DQ_ROWS);
  const int lane_at = WHOLE ? 0 : (threadIdx.x & 31) * E;                    // (ragged: the whole warp goes round, or none of it)
  for (int d0 = (blockIdx.y * lanes + t) * E - lane_at; d0 < dim; d0 += gridDim.y * lanes * E) {
    const int d = d0 + lane_at;
    uint2 u[DQ_ROWS];
    float s[DQ_ROWS];
#pragma unroll
    for (int j = 0; j < DQ_ROWS; ++j) {
      const long long row = row0 + (j < n ? j : 0) * per;                    // (rows past the last read the first again)
      if (n > 0) {
        if (WHOLE || d + E <= dim) {
          if constexpr (E == 8) u[j] = *reinterpret_cast<const uint2*>(q + row * q_rs + d);
          else u[j].x = *reinterpret_cast<const uint32_t*>(q + row * q_rs + d);
        } else {
          u[j] = make_uint2(0u, 0u);
          for (int i = 0; d + i < dim; ++i) (i < 4 ? u[j].x : u[j].y) |= (uint32_t)(uint8_t)q[row * q_rs + d + i] << (8 * (i % 4));
        }
        s[j] = scale[row];
      }
    }
#pragma unroll
    for (int j = 0; j < DQ_ROWS; ++j) {
      if (j >= n) break;
      float v[E];
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = (float)(int8_t)((i < 4 ? u[j].x : u[j].y) >> (8 * (i % 4))) * s[j];
      T* o = out + (row0 + j * per) * out_rs;
      if constexpr (WHOLE) st_chunk<T, E>(o + d, v);
      else {
        const int lane = threadIdx.x & 31, left = min(dim - d0, 32 * E);           // the warp's elements d0 ...
        T* mine = seg[threadIdx.x >> 5];
        o += d0;
#pragma unroll
        for (int c = 0; c < E * (int)sizeof(T) / 16; ++c) {
          constexpr int V = 16 / (int)sizeof(T);
          float part[V];
#pragma unroll
          for (int i = 0; i < V; ++i) part[i] = v[c * V + i];
          st_chunk<T, V>(mine + lane * E + c * V, part);
        }
        __syncwarp();
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int c = 0; c < E; ++c)
            if (lane + 32 * c < left) o[lane + 32 * c] = mine[lane + 32 * c];
        } else {                                                             // (a row may start between two words)
          const int off = (int)((reinterpret_cast<uintptr_t>(o) >> 1) & 1);
#pragma unroll
          for (int c = 0; c < E / 2 + 1; ++c) {
            const int i = 2 * lane - off + 64 * c;
            if (i >= left) break;
            if (i >= 0 && i + 1 < left) *reinterpret_cast<__nv_bfloat162*>(o + i) = __halves2bfloat162(mine[i], mine[i + 1]);
            else if (i >= 0) o[i] = mine[i];
            else o[0] = mine[0];
          }
        }
        __syncwarp();
      }
    }
  }
}

}  // namespace

static bool known_dtype(int32_t dtype) { return dtype == CODA_F32 || dtype == CODA_BF16; }
// The addresses (or nulls) lie on boundaries of elements of that size: any other access would end the context.
template <typename... P> static bool on_elements(uintptr_t bytes, const P*... p) { return (((uintptr_t)p | ... | 0) % bytes) == 0; }
static uintptr_t size_of(int32_t dtype) { return dtype == CODA_F32 ? 4 : 2; }

extern "C" int coda_b200_add_rms_norm(int32_t dtype, int64_t rows, int32_t dim, const void* x, int64_t x_rs,
                                      const void* residual, int64_t res_rs, const void* weight, float eps,
                                      void* sum, int64_t sum_rs, void* y, int64_t y_rs,
                                      int8_t* q, int64_t q_rs, float* scale, coda_stream_t stream) {
  CODA_REQUIRE(known_dtype(dtype) && rows >= 0 && dim > 0, CODA_ERR_ARG, "add_rms_norm: dtype, rows or dim invalid");
  CODA_REQUIRE(rows <= 0x7fffffffLL && dim <= 1 << 30, CODA_ERR_LIMIT, "add_rms_norm: more than 2^31 - 1 rows, or rows longer than 2^30");
  if (rows == 0) return CODA_OK;
  CODA_REQUIRE(x && weight && (residual == nullptr) == (sum == nullptr), CODA_ERR_ARG,
               "add_rms_norm: null pointer (sum and residual are given together)");
  CODA_REQUIRE(on_elements(size_of(dtype), x, residual, weight, sum, y) && on_elements(4, scale), CODA_ERR_ARG,
               "add_rms_norm: tensors must start on a boundary of their elements");
  CODA_REQUIRE((y != nullptr) != (q != nullptr) && (q != nullptr) == (scale != nullptr), CODA_ERR_ARG,
               "add_rms_norm: give either y, or q and scale");
  CODA_REQUIRE(rows == 1 || ((sum == nullptr || sum_rs >= dim) && (y == nullptr || y_rs >= dim) && (q == nullptr || q_rs >= dim)), CODA_ERR_ARG,
               "add_rms_norm: rows of an output overlap");
  CODA_REQUIRE(eps > 0.f, CODA_ERR_ARG, "add_rms_norm: eps must be positive");
  RowsParams p{rows, dim, x, x_rs, residual, res_rs, weight, eps, sum, sum_rs, y, y_rs, q, q_rs, scale};
  return dtype == CODA_F32 ? dispatch_rows<float>(p, (cudaStream_t)stream) : dispatch_rows<bf16>(p, (cudaStream_t)stream);
}

extern "C" int coda_b200_quantize_rows(int32_t dtype, int64_t rows, int32_t dim, const void* x, int64_t x_rs,
                                       int8_t* q, int64_t q_rs, float* scale, coda_stream_t stream) {
  CODA_REQUIRE(known_dtype(dtype) && rows >= 0 && dim > 0, CODA_ERR_ARG, "quantize_rows: dtype, rows or dim invalid");
  CODA_REQUIRE(rows <= 0x7fffffffLL && dim <= 1 << 30, CODA_ERR_LIMIT, "quantize_rows: more than 2^31 - 1 rows, or rows longer than 2^30");
  if (rows == 0) return CODA_OK;
  CODA_REQUIRE(x && q && scale, CODA_ERR_ARG, "quantize_rows: null pointer");
  CODA_REQUIRE(on_elements(size_of(dtype), x) && on_elements(4, scale), CODA_ERR_ARG, "quantize_rows: tensors must start on a boundary of their elements");
  CODA_REQUIRE(rows == 1 || q_rs >= dim, CODA_ERR_ARG, "quantize_rows: rows of q overlap");
  RowsParams p{rows, dim, x, x_rs, nullptr, 0, nullptr, 0.f, nullptr, 0, nullptr, 0, q, q_rs, scale};
  return dtype == CODA_F32 ? dispatch_rows<float>(p, (cudaStream_t)stream) : dispatch_rows<bf16>(p, (cudaStream_t)stream);
}

template <typename T>
static int launch_dequantize(int64_t rows, int32_t dim, const int8_t* q, int64_t q_rs, const float* scale, T* out, int64_t out_rs,
                             cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool whole = dim % V == 0 && (uintptr_t)out % 16 == 0 && out_rs % V == 0;
  const long long chunks = whole ? dim / V : ((long long)dim + 255) / 256 * 32;             // (ragged rows: whole warps)
  long long lanes = chunks < 256 ? chunks : 256;
  if (!whole) while (256 % lanes != 0) lanes += 32;
  const int at_once = whole ? 8 : 4;
  const long long per = 256 / lanes * at_once, across = (chunks + lanes - 1) / lanes;
  const dim3 grid((unsigned)((rows + per - 1) / per), (unsigned)(across < 65535 ? across : 65535));
  const auto kernel = whole ? dequantize_rows_kernel<T, V, true, 8> : dequantize_rows_kernel<T, 8, false, 4>;
  const cudaError_t e = coda_launch_chained(kernel, grid, dim3(256), 0, s, 1, (long long)rows, (int)dim, q, (long long)q_rs, scale, out,
                                            (long long)out_rs, (int)lanes);
  if (e != cudaSuccess) { coda_set_error("dequantize_rows: %s", cudaGetErrorString(e)); cudaGetLastError(); return CODA_ERR_LAUNCH; }
  return CODA_OK;
}

extern "C" int coda_b200_dequantize_rows(int32_t dtype, int64_t rows, int32_t dim, const int8_t* q, int64_t q_rs,
                                         const float* scale, void* out, int64_t out_rs, coda_stream_t stream) {
  CODA_REQUIRE(known_dtype(dtype) && rows >= 0 && dim > 0, CODA_ERR_ARG, "dequantize_rows: dtype, rows or dim invalid");
  CODA_REQUIRE(rows <= 0x7fffffffLL && dim <= 1 << 30, CODA_ERR_LIMIT, "dequantize_rows: more than 2^31 - 1 rows, or rows longer than 2^30");
  if (rows == 0) return CODA_OK;
  CODA_REQUIRE(q && scale && out, CODA_ERR_ARG, "dequantize_rows: null pointer");
  CODA_REQUIRE(on_elements(size_of(dtype), out) && on_elements(4, scale), CODA_ERR_ARG, "dequantize_rows: tensors must start on a boundary of their elements");
  CODA_REQUIRE((uintptr_t)q % 8 == 0 && q_rs % 8 == 0 && q_rs >= dim && out_rs >= dim, CODA_ERR_ARG,
               "dequantize_rows: rows of q must start on 8-byte boundaries, rows must not overlap");
  return dtype == CODA_F32 ? launch_dequantize<float>(rows, dim, q, q_rs, scale, (float*)out, out_rs, (cudaStream_t)stream)
                           : launch_dequantize<bf16>(rows, dim, q, q_rs, scale, (bf16*)out, out_rs, (cudaStream_t)stream);
}
