// Distillation from a teacher's top logits, for f32, bf16 and f16 logits: what the teacher stores (ofb_top_logits), and the student's loss
// against it with its gradient (ofb_distill_fwd / ofb_distill_bwd).  All three are bound by reading the logits: a row is cut into 16-byte
// chunks that are aligned in memory (rows of an odd number of classes start anywhere: the chunks are counted from the aligned address
// below the row, the first and the last are read element by element), each thread streams chunks and keeps a running maximum and sum.
//
// With y = z / tau over the V classes, the K stored (class, value) pairs of a row and t = value / tau:
//   L = logsumexp(t, rest)      p_k = exp(t_k - L)     p_r = exp(rest - L)
//   q = softmax(y)              q_r = sum of q over the classes that are not stored
//   loss = tau^2 [ sum_k p_k (log p_k - log q_{class k}) + p_r (log p_r - log q_r) ]
//   d loss / d z_j = tau (q_j - sum of the p_k of class j)    for a stored class
//                  = tau q_j (1 - p_r / q_r) = tau exp(y_j - m_t) (q_r - p_r) / s_t   for the others
// where m_t and s_t are the maximum of y and the sum of exp(y - m_t) over the classes that are NOT stored: they are summed apart (a bit per
// class in LDS says which is stored), so that log q_r and the small tail gradients do not come out of a difference of nearly equal sums.
// Exponentials are exp2 of (z - m) log2 e / tau with m in z's own units: exactly 0 at the maximum, and rounded relative to the distance from it, whatever the
// logits' size is.  (One fma of z with -m log2 e / tau instead leaves the rounding of that product there: 2^103 at bf16's lowest value.)
#include "hformat.h"

#define DS_F32 0
#define DS_BF16 1
#define DS_F16 2
#define DS_SEG 131072             /* classes of a segment at most: 16 KB of bits */
#define DS_THREADS 256
#define DS_KMAX 1024
#define DS_STATS 8                /* floats kept per row: m_t, kappa, m, 1/s, m_teacher, 1/s_teacher, used, 0 */
#define TL_CAP 4096               /* candidates of a row or segment that are ranked at once */
#define TL_THREADS 1024
#define TL_SMALL 256              /* threads for lists of up to TL_SMALL / 2 (1024 x 100003 bf16, 64 kept: 90 us, 1024 threads 99 us, all else alike) */

namespace {

typedef __bf16 ds_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 ds_bf16x2 __attribute__((ext_vector_type(2)));

template <int DT> struct ds_type { static constexpr int CH = 8, ES = 2; typedef unsigned short raw; };
template <> struct ds_type<DS_F32> { static constexpr int CH = 4, ES = 4; typedef float raw; };

template <int DT>
__device__ __forceinline__ float ds_value(typename ds_type<DT>::raw r) {
  if constexpr (DT == DS_F32) return r;
  else if constexpr (DT == DS_BF16) return __uint_as_float((unsigned)r << 16);
  else return (float)__builtin_bit_cast(_Float16, r);
}
template <int DT>
__device__ __forceinline__ typename ds_type<DT>::raw ds_raw(float x) {
  if constexpr (DT == DS_F32) return x;
  else if constexpr (DT == DS_BF16) return __builtin_bit_cast(unsigned short, (__bf16)x);
  else return __builtin_bit_cast(unsigned short, (_Float16)x);
}

// a row of V classes as aligned 16-byte chunks: element u = class + mis, chunk c = elements c CH .. c CH + CH - 1
template <int DT>
struct ds_row {
  const char* base;               // aligned address at or below the row
  int mis, end;                   // the row's elements are mis .. end - 1
  __device__ __forceinline__ ds_row(const void* x, int64_t row, int V) {
    const char* p = (const char*)x + row * V * ds_type<DT>::ES;
    mis = (int)((uintptr_t)p & 15) / ds_type<DT>::ES;
    base = p - mis * ds_type<DT>::ES;
    end = mis + V;
  }
  __device__ __forceinline__ int chunks() const { return (end + ds_type<DT>::CH - 1) / ds_type<DT>::CH; }
  __device__ __forceinline__ bool whole(int c) const { return c * ds_type<DT>::CH >= mis && (c + 1) * ds_type<DT>::CH <= end; }
  __device__ __forceinline__ bool has(int c, int i) const { const int u = c * ds_type<DT>::CH + i; return u >= mis && u < end; }
  __device__ __forceinline__ uint4 fetch(int c) const { return *reinterpret_cast<const uint4*>(base + (int64_t)c * 16); }
  static __device__ __forceinline__ void unpack(uint4 v, float (&x)[ds_type<DT>::CH]) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < ds_type<DT>::CH; ++i) {
      if constexpr (DT == DS_F32) x[i] = __uint_as_float(w[i]);
      else if constexpr (DT == DS_BF16) x[i] = __uint_as_float((i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
      else x[i] = (i & 1) ? ofb_f16_hi(w[i >> 1]) : ofb_f16_lo(w[i >> 1]);
    }
  }
  // runs f(chunk, values) over chunks c0 + thread, c0 + thread + THREADS, ...: `fill` stands where a chunk has no class.  Four chunks at a time
  // are loaded and handed over as one array (element i is of chunk + i / CH * THREADS): loads in flight, and one rescaling of a running sum for
  // all of them (2048 x 100003 bf16, forward of the loss: 158 us a chunk at a time, 135 us with four loads in flight, 130 us like this).  Not
  // TOGETHER: one chunk after the other, four loads in flight all the same (the backward, whose results would take the registers of a second
  // workgroup: 163 against 171 us).  Only the row's first and last chunk can be partial: they are left to the end.
  template <int THREADS, bool TOGETHER = true, typename F>
  __device__ __forceinline__ void each(int c0, int c1, float fill, F f) const {
    constexpr int CH = ds_type<DT>::CH;
    int a0 = c0, a1 = c1;
    if (a0 < a1 && !whole(a0)) ++a0;
    if (a0 < a1 && !whole(a1 - 1)) --a1;
    int c = a0 + threadIdx.x;
    for (; c + 3 * THREADS < a1; c += 4 * THREADS) {
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fetch(c + j * THREADS);
      if constexpr (TOGETHER) {
        float x[4 * CH];
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack(v[j], *reinterpret_cast<float(*)[CH]>(x + j * CH));
        f(c, x);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x[CH];
          unpack(v[j], x);
          f(c + j * THREADS, x);
        }
      }
    }
    for (; c < a1; c += THREADS) {
      float x[CH];
      unpack(fetch(c), x);
      f(c, x);
    }
    c = threadIdx.x == 0 ? c0 : c1 - 1;                       // the partial ones: thread 0 and thread 1
    if (threadIdx.x < 2 && c < c1 && !whole(c) && (threadIdx.x == 0 || c > c0 || whole(c0))) {
      float x[CH];
      load(c, x, fill);
      f(c, x);
    }
  }
  // a partial chunk's values; `fill` where there is no class
  __device__ __forceinline__ void load(int c, float (&x)[ds_type<DT>::CH], float fill) const {
    constexpr int CH = ds_type<DT>::CH;
    const char* p = base + (int64_t)c * 16;
    {
#pragma unroll
      for (int i = 0; i < CH; ++i) x[i] = has(c, i) ? ds_value<DT>(reinterpret_cast<const typename ds_type<DT>::raw*>(p)[i]) : fill;
    }
  }
};

// running maximum m and sum of exp2((x - m) c)
struct ds_sum {
  float m = -INFINITY, s = 0.f;
  template <int CH>
  __device__ __forceinline__ void add(const float (&x)[CH], float c) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < CH; ++i) top = fmaxf(top, x[i]);
    if (top > m) {                                            // (-inf alone: nothing to add; NaN: added below, the sum becomes NaN)
      s *= __builtin_amdgcn_exp2f((m - top) * c);
      m = top;
    }
    const float mu = m > -INFINITY ? m : 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) s += __builtin_amdgcn_exp2f((x[i] - mu) * c);
  }
  __device__ __forceinline__ void join(float m2, float s2, float c) {
    const float n = fmaxf(m, m2), mu = n > -INFINITY ? n : 0.f;
    s = s * __builtin_amdgcn_exp2f((m - mu) * c) + s2 * __builtin_amdgcn_exp2f((m2 - mu) * c);
    m = n;
  }
};

__device__ __forceinline__ double ds_wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// workgroup reductions; every thread gets the result (red: one word per wave, free before and after)
template <int THREADS>
__device__ __forceinline__ double ds_total(double v, double* red) {
  v = ds_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / 64; ++i) v += red[i];
  return v;
}
template <int THREADS>
__device__ __forceinline__ ds_sum ds_join(ds_sum a, float c, float* redm, float* reds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(a.m, o, 64), s2 = __shfl_xor(a.s, o, 64);
    const float n = fmaxf(a.m, m2), mu = n > -INFINITY ? n : 0.f;      // (symmetric: every lane computes the same)
    const float x = a.s * __builtin_amdgcn_exp2f((a.m - mu) * c), y = s2 * __builtin_amdgcn_exp2f((m2 - mu) * c);
    a.s = x + y;
    a.m = n;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { redm[threadIdx.x >> 6] = a.m; reds[threadIdx.x >> 6] = a.s; }
  __syncthreads();
  ds_sum r;
  r.m = redm[0];
  r.s = reds[0];
#pragma unroll
  for (int i = 1; i < THREADS / 64; ++i) r.join(redm[i], reds[i], c);
  return r;
}

struct ds_args {
  const void *z, *values, *indices;
  const float* rest;
  float *stats, *part, *row_loss;
  void* dz;
  const float* up;
  int64_t R;
  int V, K, segs, idx64, up_rows;
  float c, tau, grad_scale;
};

// the class of entry k of a row, or -1: outside 0 .. V - 1, or a value of -inf
template <int DT>
__device__ __forceinline__ int ds_class(const ds_args& a, int64_t row, int k, float& value) {
  const int64_t at = row * a.K + k;
  const int64_t i = a.idx64 ? ((const int64_t*)a.indices)[at] : (int64_t)((const int32_t*)a.indices)[at];
  value = ds_value<DT>(((const typename ds_type<DT>::raw*)a.values)[at]);
  return (i < 0 || i >= a.V || value == -INFINITY) ? -1 : (int)i;
}

// whether no entry before k has class i (cls: 16-byte aligned, padded to a multiple of four)
__device__ __forceinline__ bool ds_first(const int* cls, int k, int i) {
  bool first = true;
  for (int e = 0; e < k; e += 4) {
    const int4 o = *reinterpret_cast<const int4*>(&cls[e]);
    first &= o.x != i;
    first &= o.y != i || e + 1 >= k;
    first &= o.z != i || e + 2 >= k;
    first &= o.w != i || e + 3 >= k;
  }
  return first;
}

// a row's entries in LDS: class (or -1), stored value, the student's logit, and the same or -inf where an earlier entry has the class (the first
// stands for it in sums over the classes)
struct ds_entries {
  int* cls;
  float *t, *y, *own;
  __device__ __forceinline__ ds_entries(int* at, int K) : cls(at), t((float*)at + ((K + 3) & ~3)), y(t + ((K + 3) & ~3)), own(y + ((K + 3) & ~3)) {}
  static constexpr int words(int K) { return 4 * ((K + 3) & ~3); }
};
template <int DT>
__device__ __forceinline__ int ds_load_entries(const ds_args& a, int64_t row, ds_entries e) {      // -> how many classes there are
  for (int k = threadIdx.x; k < ((a.K + 3) & ~3); k += DS_THREADS) {
    float v = 0.f;
    const int i = k < a.K ? ds_class<DT>(a, row, k, v) : -1;
    e.cls[k] = i;
    e.t[k] = v;
    e.y[k] = i < 0 ? 0.f : ds_value<DT>(((const typename ds_type<DT>::raw*)a.z)[row * a.V + i]);
  }
  __syncthreads();
  int classes = 0;
  for (int k0 = 0; k0 < a.K; k0 += DS_THREADS) {
    const int k = k0 + threadIdx.x;
    const bool first = k < a.K && e.cls[k] >= 0 && ds_first(e.cls, k, e.cls[k]);
    if (k < a.K) e.own[k] = first ? e.y[k] : -INFINITY;
    classes += __syncthreads_count(first);
  }
  return classes;
}

// The row's loss and what the backward needs, from (m_t, s_t) of the classes that are not stored: one wave (the other waves of the workgroup are
// done, and nothing waits for a barrier).  The sums over the stored classes are in 64 bits: the loss is a difference of logarithms of the size of log V.
__device__ void ds_finish(const ds_args& a, int64_t row, ds_sum tail, ds_entries e, int classes) {
  const int lane = threadIdx.x & 63;
  float mt = -INFINITY, m = tail.m;
  for (int k = lane; k < a.K; k += 64) {
    if (e.cls[k] < 0) continue;
    mt = fmaxf(mt, e.t[k]);
    m = fmaxf(m, e.y[k]);
  }
  mt = ofb_wave_max(mt);
  m = ofb_wave_max(m);
  const bool any = classes > 0, all = classes >= a.V;                              // every class is stored: there is no rest
  const double r2 = (a.rest && !all) ? (double)a.rest[row] * 1.44269504088896340736 : -INFINITY;
  mt = fmaxf(mt, (float)(r2 / (double)a.c));
  const float mtu = mt > -INFINITY ? mt : 0.f, mu = m > -INFINITY ? m : 0.f;
  double st = 0.0, s = 0.0;
  for (int k = lane; k < a.K; k += 64) {
    if (e.cls[k] < 0) continue;
    st += (double)__builtin_amdgcn_exp2f((e.t[k] - mtu) * a.c);
    s += (double)__builtin_amdgcn_exp2f((e.own[k] - mu) * a.c);
  }
  const float er = __builtin_amdgcn_exp2f((float)(r2 - (double)mtu * (double)a.c)), et = tail.s > 0.f ? tail.s * __builtin_amdgcn_exp2f((tail.m - mu) * a.c) : tail.s;
  st = ds_wave_sum(st) + (double)er;
  s = ds_wave_sum(s) + (double)et;
  const double c = (double)a.c, lt = log2(st), ls = log2(s), ci = 1.0 / st;      // (logarithms relative to the maxima: log V does not survive beside 1e38)
  double loss = 0.0;
  for (int k = lane; k < a.K; k += 64) {
    if (e.cls[k] < 0) continue;
    const double p = (double)__builtin_amdgcn_exp2f((e.t[k] - mtu) * a.c) * ci;
    loss += p * (((double)e.t[k] - (double)mtu) * c - lt - ((double)e.y[k] - (double)mu) * c + ls);
  }
  loss = ds_wave_sum(loss);
  const double pr = (double)er * ci;
  if (pr > 0.0) loss += pr * (r2 - (double)mtu * c - lt - (((double)tail.m - (double)mu) * c + log2((double)tail.s) - ls));
  if (lane == 0) {
    float* o = a.stats + row * DS_STATS;
    o[0] = tail.m > -INFINITY ? tail.m : 0.f;
    o[1] = tail.s == 0.f ? 0.f : (float)(((double)et / s - pr) / (double)tail.s);
    o[2] = mu;
    o[3] = (float)(1.0 / s);
    o[4] = mtu;
    o[5] = (float)ci;
    o[6] = any ? 1.f : 0.f;
    o[7] = 0.f;
    a.row_loss[row] = any ? (float)(loss * 0.69314718055994530942 * (double)a.tau * (double)a.tau) : 0.f;
  }
}

template <int DT, bool WHOLE>      // WHOLE: one segment a row, which also finishes it
__global__ __launch_bounds__(DS_THREADS) void distill_fwd_kernel(ds_args a) {
  constexpr int CH = ds_type<DT>::CH;
  // a bit per class of the segment and the entries: as much LDS as they take, so that eight workgroups share a CU
  extern __shared__ __attribute__((aligned(16))) int lds[];
  const ds_entries e(lds, a.K);
  unsigned* bits = reinterpret_cast<unsigned*>(lds + ds_entries::words(a.K));
  __shared__ float redf[8];
  const int64_t row = blockIdx.x / a.segs;
  const int seg = blockIdx.x % a.segs;
  const ds_row<DT> r(a.z, row, a.V);
  const int nc = r.chunks(), per = (nc + a.segs - 1) / a.segs, c0 = min(nc, seg * per), c1 = min(nc, c0 + per);
  for (int i = threadIdx.x; i < (c1 - c0) * CH / 32 + 1; i += DS_THREADS) bits[i] = 0u;
  int classes = 0;
  if constexpr (WHOLE) classes = ds_load_entries<DT>(a, row, e);
  __syncthreads();
  for (int k = threadIdx.x; k < a.K; k += DS_THREADS) {
    float v;
    const int i = WHOLE ? e.cls[k] : ds_class<DT>(a, row, k, v), u = i + r.mis - c0 * CH;
    if (i >= 0 && u >= 0 && u < (c1 - c0) * CH) atomicOr(&bits[u >> 5], 1u << (u & 31));
  }
  __syncthreads();
  ds_sum sum;
  r.template each<DS_THREADS>(c0, c1, -INFINITY, [&](int c, auto& x) {
    constexpr int N = sizeof(x) / 4, B = N / CH;
    unsigned b[B], any = 0u;
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int u = (c + j * DS_THREADS - c0) * CH;
      b[j] = (bits[u >> 5] >> (u & 31)) & ((1u << CH) - 1u);
      any |= b[j];
    }
    if (any) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (b[i / CH] >> (i % CH) & 1) x[i] = -INFINITY;
    }
    sum.add<N>(x, a.c);
  });
  sum = ds_join<DS_THREADS>(sum, a.c, redf, redf + 4);
  if constexpr (WHOLE) {
    if (threadIdx.x < 64) ds_finish(a, row, sum, e, classes);
  } else if (threadIdx.x == 0) {
    a.part[2 * blockIdx.x] = sum.m;
    a.part[2 * blockIdx.x + 1] = sum.s;
  }
}

template <int DT>
__global__ __launch_bounds__(DS_THREADS) void distill_finish_kernel(ds_args a) {
  extern __shared__ __attribute__((aligned(16))) int lds[];
  const ds_entries e(lds, a.K);
  __shared__ float redf[8];
  const int64_t row = blockIdx.x;
  ds_sum sum;
  for (int i = threadIdx.x; i < a.segs; i += DS_THREADS) sum.join(a.part[2 * (row * a.segs + i)], a.part[2 * (row * a.segs + i) + 1], a.c);
  const int classes = ds_load_entries<DT>(a, row, e);
  sum = ds_join<DS_THREADS>(sum, a.c, redf, redf + 4);
  if (threadIdx.x < 64) ds_finish(a, row, sum, e, classes);
}

__global__ __launch_bounds__(DS_THREADS) void distill_reduce_kernel(const float* __restrict__ row_loss, int64_t R, double scale, float* __restrict__ out) {
  __shared__ double red[4];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < R; i += DS_THREADS) s += (double)row_loss[i];
  s = ds_total<DS_THREADS>(s, red);
  if (threadIdx.x == 0) out[0] = (float)(s * scale);
}

// every class of the segment is written as one that is not stored; then the stored ones are written over (one thread each)
template <int DT>
__global__ __launch_bounds__(DS_THREADS) void distill_bwd_kernel(ds_args a) {
  constexpr int CH = ds_type<DT>::CH;
  typedef typename ds_type<DT>::raw raw;
  __shared__ __attribute__((aligned(16))) int cls[DS_KMAX];
  __shared__ float prob[DS_KMAX];
  const int64_t row = blockIdx.x / a.segs;
  const int seg = blockIdx.x % a.segs;
  const ds_row<DT> r(a.z, row, a.V);
  const int nc = r.chunks(), per = (nc + a.segs - 1) / a.segs, c0 = min(nc, seg * per), c1 = min(nc, c0 + per);
  const float* st = a.stats + row * DS_STATS;
  const float mt = st[0], m = st[2], is = st[3], mk = st[4], ik = st[5];
  const bool used = st[6] != 0.f;
  const float g = a.up[a.up_rows ? row : 0] * a.grad_scale, kappa = st[1] * g;
  char* out = (char*)a.dz + (row * a.V - r.mis) * (int64_t)ds_type<DT>::ES;
  r.template each<DS_THREADS, false>(c0, c1, 0.f, [&](int c, float (&x)[CH]) {
#pragma unroll
    for (int i = 0; i < CH; ++i) x[i] = used ? __builtin_amdgcn_exp2f((x[i] - mt) * a.c) * kappa : 0.f;
    char* p = out + (int64_t)c * 16;
    if (r.whole(c)) {
      if constexpr (DT == DS_F32) {
        *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
      } else {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (DT == DS_BF16) { ofb_f32x2 v = {x[2 * i], x[2 * i + 1]}; w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, ds_bf16x2)); }
          else w[i] = ofb_pk_f16(x[2 * i], x[2 * i + 1]);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (r.has(c, i)) reinterpret_cast<raw*>(p)[i] = ds_raw<DT>(x[i]);
    }
  });
  if (!used) return;
  for (int k = threadIdx.x; k < ((a.K + 3) & ~3); k += DS_THREADS) {
    float v = 0.f;
    cls[k] = k < a.K ? ds_class<DT>(a, row, k, v) : -1;
    prob[k] = cls[k] < 0 ? 0.f : __builtin_amdgcn_exp2f((v - mk) * a.c) * ik;
  }
  __syncthreads();                                             // ... and the stores above come before those below
  for (int k = threadIdx.x; k < a.K; k += DS_THREADS) {
    const int i = cls[k], u = i + r.mis;
    if (i < 0 || u < c0 * CH || u >= c1 * CH) continue;
    if (!ds_first(cls, k, i)) continue;
    float p = prob[k];
    for (int e = (k + 1) & ~3; e < a.K; e += 4) {
      const int4 o = *reinterpret_cast<const int4*>(&cls[e]);
      if (o.x == i && e > k) p += prob[e];
      if (o.y == i && e + 1 > k) p += prob[e + 1];
      if (o.z == i && e + 2 > k) p += prob[e + 2];
      if (o.w == i && e + 3 > k) p += prob[e + 3];
    }
    const int64_t at = row * a.V + i;
    const float q = __builtin_amdgcn_exp2f((ds_value<DT>(((const raw*)a.z)[at]) - m) * a.c) * is;
    ((raw*)a.dz)[at] = ds_raw<DT>((q - p) * g);
  }
}

// ------------------------------------------------------------------------------------------------------------------
// top logits
// ------------------------------------------------------------------------------------------------------------------
// An element's rank key: its value's bits made to order like unsigned integers (NaN above everything, -0 as +0), then the complement of its
// class, so that ties go to the lowest class and no two keys are equal.  0 is no element's key.
__device__ __forceinline__ unsigned tl_key(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float tl_float(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

struct tl_args {
  const void* z;
  void* values;
  int32_t* indices;
  float* rest;
  unsigned long long* cand;        // [R][segs][K]
  float* part;                     // [R][segs][2]
  int64_t R;
  int V, K, segs;
  float c;
};

// ranks n distinct keys in LDS by counting the greater ones; the first K leave through `out(rank, key)`, the values of the others are added
// to `sum` in the order of their ranks
template <int THREADS, typename OUT>
__device__ __forceinline__ ds_sum tl_rank(unsigned long long* list, float* left, int n, int K, float c, ds_sum sum, OUT out) {
  if (threadIdx.x == 0 && (n & 1)) list[n] = 0ull;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long k = list[i];
    int rank = 0;
    for (int e = 0; e < n; e += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&list[e]);
      rank += (o.x > k) + (o.y > k);
    }
    if (rank < K) out(rank, k);
    else left[rank - K] = tl_float((unsigned)(k >> 32));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n - K; i += THREADS) {
    const float x[1] = {left[i]};
    sum.add<1>(x, c);
  }
  return sum;
}

// log-sum-exp; of finite logits it stays finite (the type's lowest value over a temperature of 1)
__device__ __forceinline__ float tl_rest(ds_sum sum, float c) {
  const float r = (float)(((double)sum.m * (double)c + log2((double)sum.s)) * 0.69314718055994530942);
  return fabsf(sum.m) < INFINITY ? fminf(fmaxf(r, -3.402823466e38f), 3.402823466e38f) : r;
}

template <int DT, int THREADS, bool WHOLE>
__global__ __launch_bounds__(THREADS, 4) void top_logits_kernel(tl_args a) {
  constexpr int CH = ds_type<DT>::CH;
  // Small workgroups: half the list and at most 128 registers, so that four share a CU (1024 rows are then one round of the chip: 1024 x 100003
  // bf16, 64 kept: 90 us with the whole list and as many registers as the compiler likes, 75 us so; 78 us with today's exponentials).
  constexpr int CAP = THREADS == TL_SMALL ? TL_CAP / 2 : TL_CAP;
  __shared__ __attribute__((aligned(16))) unsigned long long list[CAP + 2];
  __shared__ float left[CAP];
  __shared__ float redm[THREADS / 64], reds[THREADS / 64];
  __shared__ int count;
  __shared__ unsigned bound;
  unsigned* tops = reinterpret_cast<unsigned*>(left);
  const int64_t row = blockIdx.x / a.segs;
  const int seg = blockIdx.x % a.segs;
  const ds_row<DT> r(a.z, row, a.V);
  const int nc = r.chunks(), per = (nc + a.segs - 1) / a.segs, c0 = min(nc, seg * per), c1 = min(nc, c0 + per);
  const int have = max(0, min(r.end, c1 * CH) - max(r.mis, c0 * CH)), K = min(a.K, have);

  // A bound for the K-th largest element: the K-th largest of the threads' own maxima - K different elements are at least that large, and
  // hardly more than K are when the threads' elements are no sorted run.  (NaN are left out of the maxima; they pass the bound below.)
  float top = -INFINITY;
  bool any = false;
  r.template each<THREADS>(c0, c1, -INFINITY, [&](int, auto& x) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(x) / 4); ++i) top = fmaxf(top, x[i]);
    any = true;
  });
  if (threadIdx.x == 0) count = 0;
  tops[threadIdx.x] = any ? tl_key(top) : 0u;
  __syncthreads();
  if (threadIdx.x < 64) {                                      // one wave bisects the upper 20 bits of the maxima's keys, rounded down
    unsigned v[THREADS / 64], found = 0u;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) v[i] = tops[threadIdx.x + 64 * i];
    for (int bit = 31; bit >= 12; --bit) {
      const unsigned probe = found | (1u << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < THREADS / 64; ++i) n += __popcll(__ballot(v[i] >= probe));
      if (n >= K) found = probe;
    }
    if (threadIdx.x == 0) bound = found;
  }
  __syncthreads();
  // no NaN is less than the bound, and nothing is where the bound is no number: too few threads have elements
  const float least = tl_float(bound);
  ds_sum sum;
  r.template each<THREADS>(c0, c1, -INFINITY, [&](int c, auto& x) {
    constexpr int N = sizeof(x) / 4;
    bool hit = false;
#pragma unroll
    for (int i = 0; i < N; ++i) hit |= !(x[i] < least);
    if (hit) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at_c = c + i / CH * THREADS;
        if (!(x[i] < least) && r.has(at_c, i % CH)) {
          const int at = atomicAdd(&count, 1);
          if (at < CAP) list[at] = ((unsigned long long)tl_key(x[i]) << 32) | (unsigned)~(unsigned)(at_c * CH + i % CH - r.mis);
          x[i] = -INFINITY;
        }
      }
    }
    sum.add<N>(x, a.c);
  });
  __syncthreads();
  int n = count;
  if (n > CAP) {
    // many equal elements, or a sorted run: the K-th largest key itself, bit by bit from the top
    unsigned long long floor_key = 0ull;
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long probe = floor_key | (1ull << bit);
      int k = 0;
      r.template each<THREADS>(c0, c1, 0.f, [&](int c, auto& x) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(x) / 4); ++i) {
          const int at_c = c + i / CH * THREADS;
          k += r.has(at_c, i % CH) && (((unsigned long long)tl_key(x[i]) << 32) | (unsigned)~(unsigned)(at_c * CH + i % CH - r.mis)) >= probe;
        }
      });
      __syncthreads();
      if (threadIdx.x == 0) count = 0;
      __syncthreads();
      if (k) atomicAdd(&count, k);
      __syncthreads();
      if (count >= K) floor_key = probe;
    }
    __syncthreads();
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    sum = ds_sum();
    r.template each<THREADS>(c0, c1, -INFINITY, [&](int c, auto& x) {
      constexpr int N = sizeof(x) / 4;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at_c = c + i / CH * THREADS;
        const unsigned long long k = ((unsigned long long)tl_key(x[i]) << 32) | (unsigned)~(unsigned)(at_c * CH + i % CH - r.mis);
        if (r.has(at_c, i % CH) && k >= floor_key) {
          list[atomicAdd(&count, 1)] = k;
          x[i] = -INFINITY;
        }
      }
      sum.add<N>(x, a.c);
    });
  }
  __syncthreads();
  n = count;
  auto leave = [&](int rank, unsigned long long k) {
    if constexpr (WHOLE) {
      const int cls = (int)~(unsigned)k;
      a.indices[row * a.K + rank] = cls;
      ((typename ds_type<DT>::raw*)a.values)[row * a.K + rank] = ((const typename ds_type<DT>::raw*)a.z)[row * a.V + cls];
    } else {
      a.cand[(int64_t)blockIdx.x * a.K + rank] = k;
    }
  };
  sum = tl_rank<THREADS>(list, left, n, K, a.c, sum, leave);
  if constexpr (!WHOLE)
    for (int i = K + threadIdx.x; i < a.K; i += THREADS) a.cand[(int64_t)blockIdx.x * a.K + i] = 0ull;
  sum = ds_join<THREADS>(sum, a.c, redm, reds);
  if (threadIdx.x == 0) {
    if constexpr (WHOLE) a.rest[row] = tl_rest(sum, a.c);
    else { a.part[2 * blockIdx.x] = sum.m; a.part[2 * blockIdx.x + 1] = sum.s; }
  }
}

template <int DT>
__global__ __launch_bounds__(TL_THREADS) void top_logits_join_kernel(tl_args a) {
  __shared__ __attribute__((aligned(16))) unsigned long long list[TL_CAP + 2];
  __shared__ float left[TL_CAP];
  __shared__ float redm[TL_THREADS / 64], reds[TL_THREADS / 64];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < a.segs * a.K; i += TL_THREADS) {
    const unsigned long long k = a.cand[row * a.segs * a.K + i];
    if (k) list[atomicAdd(&count, 1)] = k;
  }
  __syncthreads();
  const int n = count;
  ds_sum sum;
  if (threadIdx.x == 0)
    for (int i = 0; i < a.segs; ++i) sum.join(a.part[2 * (row * a.segs + i)], a.part[2 * (row * a.segs + i) + 1], a.c);
  sum = tl_rank<TL_THREADS>(list, left, n, a.K, a.c, sum, [&](int rank, unsigned long long k) {
    const int cls = (int)~(unsigned)k;
    a.indices[row * a.K + rank] = cls;
    ((typename ds_type<DT>::raw*)a.values)[row * a.K + rank] = ((const typename ds_type<DT>::raw*)a.z)[row * a.V + cls];
  });
  sum = ds_join<TL_THREADS>(sum, a.c, redm, reds);
  if (threadIdx.x == 0) a.rest[row] = tl_rest(sum, a.c);
}

int ds_es(int dtype) { return dtype == DS_F32 ? 4 : 2; }
// segments of a row: what its bits' LDS allows, and more where the rows alone leave the chip idle (at least 4096 classes each)
int ds_segments(int64_t R, int V) {
  const int64_t must = ((int64_t)V + 8 + DS_SEG - 9) / (DS_SEG - 8);
  const int64_t want = (1024 + R - 1) / R, most = V / 4096;
  const int64_t s = want < most ? want : most;
  return (int)(s > must ? s : must);
}
int tl_segments(int64_t R, int V, int K) {
  const int64_t want = (512 + R - 1) / R, most = V / 8192, room = TL_CAP / K;
  int64_t s = want < most ? want : most;
  s = s < room ? s : room;
  return (int)(s < 1 ? 1 : s);
}
int ds_check(const void* z, const void* values, const void* indices, int64_t R, int32_t V, int32_t K, float tau, int32_t dtype) {
  if (!z || !values || !indices || R < 1 || V < 1 || K < 1 || dtype < 0 || dtype > 2 || !(tau > 1e-37f) || !(tau < 3.0e38f)) return OFB_EINVAL;
  if (K > DS_KMAX || K > V || V > (1 << 30) || R >= (1 << 22)) return OFB_ELIMIT;      // (threads of a launch count in 32 bits)
  if (!ofb_aligned16(z)) return OFB_EINVAL;
  return OFB_OK;
}

}  // namespace

extern "C" int ofb_distill_segments(int64_t R, int32_t V) { return (R < 1 || V < 1) ? 0 : ds_segments(R, V); }
extern "C" int ofb_top_logits_segments(int64_t R, int32_t V, int32_t K) { return (R < 1 || V < 1 || K < 1) ? 0 : tl_segments(R, V, K); }

extern "C" int ofb_distill_fwd(const void* z, const void* values, const void* indices, int32_t idx64, const float* rest, int64_t R, int32_t V, int32_t K,
                               float tau, int32_t dtype, float* stats, float* part, float* row_loss, double loss_scale, float* loss, void* stream) {
  if (const int rc = ds_check(z, values, indices, R, V, K, tau, dtype)) return rc;
  if (!stats || !row_loss) return OFB_EINVAL;
  ds_args a = {};
  a.z = z; a.values = values; a.indices = indices; a.rest = rest; a.stats = stats; a.part = part; a.row_loss = row_loss;
  a.R = R; a.V = V; a.K = K; a.segs = ds_segments(R, V); a.idx64 = idx64; a.c = (float)(1.4426950408889634074 / (double)tau); a.tau = tau;
  if (a.segs > 1 && !part) return OFB_EINVAL;
  if (R * a.segs >= (1 << 22)) return OFB_ELIMIT;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(R * a.segs)), block(DS_THREADS);
  // (a row spans one chunk more than V classes take where it starts inside one; the last word is only cleared)
  const int ch = 16 / ds_es(dtype), nc = (V + 2 * ch - 2) / ch, lds = (ds_entries::words(K) + (nc + a.segs - 1) / a.segs * ch / 32 + 2) * 4;
#define DS_FWD(DT)                                                                                        \
  if (a.segs == 1) hipLaunchKernelGGL((distill_fwd_kernel<DT, true>), grid, block, lds, s, a);            \
  else {                                                                                                  \
    hipLaunchKernelGGL((distill_fwd_kernel<DT, false>), grid, block, lds, s, a);                          \
    hipLaunchKernelGGL((distill_finish_kernel<DT>), dim3((unsigned)R), block, ds_entries::words(K) * 4, s, a);                   \
  }
  if (dtype == DS_F32) { DS_FWD(DS_F32) } else if (dtype == DS_BF16) { DS_FWD(DS_BF16) } else { DS_FWD(DS_F16) }
  if (loss) hipLaunchKernelGGL(distill_reduce_kernel, dim3(1), block, 0, s, row_loss, R, loss_scale, loss);
  return ofb_launch_status();
}

extern "C" int ofb_distill_bwd(const void* z, const void* values, const void* indices, int32_t idx64, int64_t R, int32_t V, int32_t K, float tau,
                               int32_t dtype, const float* stats, const float* up, int32_t up_rows, float grad_scale, void* dz, void* stream) {
  if (const int rc = ds_check(z, values, indices, R, V, K, tau, dtype)) return rc;
  if (!stats || !up || !dz || !ofb_aligned16(dz)) return OFB_EINVAL;
  ds_args a = {};
  a.z = z; a.values = values; a.indices = indices; a.stats = (float*)stats; a.dz = dz; a.up = up; a.up_rows = up_rows; a.grad_scale = grad_scale;
  a.R = R; a.V = V; a.K = K; a.segs = ds_segments(R, V); a.idx64 = idx64; a.c = (float)(1.4426950408889634074 / (double)tau); a.tau = tau;
  if (R * a.segs >= (1 << 22)) return OFB_ELIMIT;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(R * a.segs)), block(DS_THREADS);
  if (dtype == DS_F32) hipLaunchKernelGGL((distill_bwd_kernel<DS_F32>), grid, block, 0, s, a);
  else if (dtype == DS_BF16) hipLaunchKernelGGL((distill_bwd_kernel<DS_BF16>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((distill_bwd_kernel<DS_F16>), grid, block, 0, s, a);
  return ofb_launch_status();
}

extern "C" int ofb_top_logits(const void* z, int64_t R, int32_t V, int32_t K, float tau, int32_t dtype, void* values, int32_t* indices, float* rest,
                              void* cand, float* part, void* stream) {
  if (const int rc = ds_check(z, values, indices, R, V, K, tau, dtype)) return rc;
  if (!rest) return OFB_EINVAL;
  tl_args a = {z, values, indices, rest, (unsigned long long*)cand, part, R, V, K, tl_segments(R, V, K), (float)(1.4426950408889634074 / (double)tau)};
  if (a.segs > 1 && (!cand || !part)) return OFB_EINVAL;
  if (R * a.segs >= (1 << 22)) return OFB_ELIMIT;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(R * a.segs));
#define TL_RUN(DT)                                                                                                        \
  if (a.segs > 1) {                                                                                                       \
    hipLaunchKernelGGL((top_logits_kernel<DT, TL_THREADS, false>), grid, dim3(TL_THREADS), 0, s, a);                      \
    hipLaunchKernelGGL((top_logits_join_kernel<DT>), dim3((unsigned)R), dim3(TL_THREADS), 0, s, a);                       \
  } else if (K <= TL_SMALL / 2) {                                                                                         \
    hipLaunchKernelGGL((top_logits_kernel<DT, TL_SMALL, true>), grid, dim3(TL_SMALL), 0, s, a);                                     \
  } else {                                                                                                                \
    hipLaunchKernelGGL((top_logits_kernel<DT, TL_THREADS, true>), grid, dim3(TL_THREADS), 0, s, a);                       \
  }
  if (dtype == DS_F32) { TL_RUN(DS_F32) } else if (dtype == DS_BF16) { TL_RUN(DS_BF16) } else { TL_RUN(DS_F16) }
  return ofb_launch_status();
}
