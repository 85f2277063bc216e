// Attention with a learned relative position bias by buckets, forward and backward, for f32, bf16 and f16 tensors:
//
//   S_ij = scale q_i . k_j + T[bucket(pos_k[j] - pos_q[i])][h],   P = softmax_j S over the keys that query i sees,   O = P V
//   D_i = dO_i . O_i,  dP = dO V^T,  dS = P (dP - D),  dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q,
//   dT[c][h] = sum over the batch and over the pairs of bucket c of dS.
//
// The bias never exists as a matrix: a pair's bucket goes by the clamped difference of two integer positions, so each head's bias is a
// vector w[difference - lo] (a few hundred floats, already times log2 e) that every workgroup gathers from the table into LDS.  Positions
// are j and i + q_offset, or come from two int32 arrays (a patch grid: y (2 w - 1) + x makes one number of two coordinates).
//
// Matrix products: v_mfma_f32_32x32x16.  bf16 and f16 operands as they are; f32 operands as two f16 planes of a power-of-two scaled copy and
// three products (hformat.h), with exponents from the maxima of the tile (Q, dO, dS) or of the head (K, V; of all heads where a pass of its own
// finds them).  Scores, softmax statistics, dS and all sums are f32 (the table's gradient sums in 64 bits); P and dS are rounded to the operand
// type for the second product: bf16 as they are, f16 with dS times a power of two that keeps it below 2^15 (and P times 2^14 for dV), f32 likewise
// in two f16 planes.  (f32 operands of any size: exponents run from 2^-113, for f32's largest value, to 2^112, where a tensor whose maximum is below 2^-97 is
// held to 2^-137.  What has to fit f32 is what f32 arithmetic forms too: scores, dP and dS.  A value keeps 22 bits, and no less than 2^-39 of the maximum behind its
// exponent: one huge key or value lowers what the rows that do not meet it keep.)
// bf16 / f16: P and dS as one term, because their rounding is of the size of the operands' own, and the result's: errors against 64 bits are 1.2 to 1.45 times those of one rounding at
// the end (bf16: 0.0021 / 0.0017 for out, 0.0024 / 0.0017 for the gradients; f16: 0.00029 / 0.00021).  As two terms (value and remainder) they are those of one rounding, and the kernels run
// one product more for each: 6007 tokens bf16, train, 1064 and 1286 us; 16 x 512 181 and 198; 4 x 1025 causal f16 187 and 205; one token over caches 94 and 101.
//
// Operand conventions (lane l, hh = l >> 5): A[row = l & 31][k = 8 hh + j], B[k = 8 hh + j][col = l & 31], accumulator register r holds
// row 8 (r >> 2) + 4 hh + (r & 3) of column l & 31.  A reduction may run over its index in any order that both operands share, so an
// accumulator feeds the next product as its B operand without leaving its registers: registers 8 s .. 8 s + 7 are the k-slots of step s,
// and the A operand is read with rows 16 s + 8 (j >> 2) + 4 hh + (j & 3) - two transposing LDS reads of four rows each.
#include "hformat.h"

#define RP_F32 0
#define RP_BF16 1
#define RP_F16 2
#define RP_THREADS 256
#define RP_TILE 128              /* queries (forward, dQ) or keys (dK dV, table gradient) of a workgroup: four waves of 32 */
#define RP_PAD 4                 /* entries of w on either side, so that four consecutive differences need one clamp */
#define RP_WMAX 4096
#define RP_PE 14                 /* f32's planes, and the backward's f16, hold P 2^14 */
#define RP_EMIN -113             /* exponents of the planes: f32's largest value times 2^-113 is below 2^15 */
#define RP_EMAX 112              /* ... and 2^-(112 + RP_PE) is still a normal number */
#define RP_ESMAX 126             /* dS is scaled by 2^RP_EMIN .. 2^126 */
#define RP_NBOUND 256            /* partial maxima of a tensor */
// A weight is exp2 of the ROUNDED score minus the row's maximum, which is a rounded score: 1 at most, and the same in every kernel.  Tiles of one bias leave
// the rounding out (one fma: the product plus bias - maximum) only where maximum and bias are at most this, in log2 units: scores are then known to 2^-14,
// and so is what the two forms differ by.  Beyond, a weight could be exp2 of half the last place of 1e9.
#define RP_PLAIN 1024.f
// Keys up to which a workgroup of the f32 forward reads its head's K and V once more for their maxima; a pass of its own over both otherwise.  Both, heads
// of 64: 128 x 197 keys, 6 heads 68 and 73 us; 32 x 256, 6 heads 26 and 31; 16 x 512, 12 heads 65.5 and 67.5; 8 x 768 75.7 and 76.6; 8 x 1024 111 and 108.
#define RP_OWN 512

namespace {

typedef __bf16 rp_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 rp_bf16x2 __attribute__((ext_vector_type(2)));
typedef short rp_s16x4 __attribute__((ext_vector_type(4)));
typedef short rp_s16x8 __attribute__((ext_vector_type(8)));
typedef rp_s16x8 rp_frag;

template <int DT> struct rp_type { static constexpr int NP = 1, ES = 2; };
template <> struct rp_type<RP_F32> { static constexpr int NP = 2, ES = 4; };

// Rows of a streamed tile of kernel 0 forward, 1 dQ, 2 dK dV, 3 dQ where workgroups are few (rp_few).  More rows are fewer barriers, until the staging
// registers or the LDS cost a workgroup, or they spill.  Measured both sides: 16-bit, d 64 (6007 tokens, 16 heads): forward 128 rows 246, 64 rows 213 us; dK dV 64 rows 553, 128 rows 521 us;
// dQ alike.  16-bit, d 128 (4 x 1025 causal, 8 heads): forward 32 rows 47, 64 rows 41 us; dK dV 87 and 68 us; dQ 89 and 119 us.  f32, d 64 (14 x 14 grid,
// B 128): 32 rows 59 / 113 / 101 us, 64 rows 87 / 165 / 101 us.
template <int DT, int DP> constexpr int rp_rows_of(int kernel) {
  constexpr int f32[4] = {32, 32, 32, 32}, narrow[4] = {64, 64, 128, 64}, wide[4] = {64, 32, 64, 64};
  return DT == RP_F32 ? f32[kernel] : DP <= 64 ? narrow[kernel] : wide[kernel];
}
template <int DT, int DP, int ROWS> struct rp_geo {
  static constexpr int NP = rp_type<DT>::NP;
  static constexpr int KB = ROWS;
  static constexpr int PITCH = DP * 2 + 16;                  // bytes of a row of one plane: 8 rows' 16-byte chunks fall into different banks
  static constexpr int PLANE = KB * PITCH;
  static constexpr int TENSOR = NP * PLANE;
  static constexpr int STAGE = 2 * TENSOR;                   // two tensors (K and V, or Q and dO)
  static constexpr int CHUNKS = KB * DP / 8;
  static constexpr int PER = (CHUNKS + RP_THREADS - 1) / RP_THREADS;
};

template <int DT>
__device__ __forceinline__ f32x16 rp_mm1(rp_frag a, rp_frag b, f32x16 c) {
  if constexpr (DT == RP_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(rp_bf16x8, a), __builtin_bit_cast(rp_bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ofb_f16x8, a), __builtin_bit_cast(ofb_f16x8, b), c, 0, 0, 0);
}
// SWAPPED: the terms in the order of the product whose A and B are this one's B and A, whose sums are then the same to the last bit
template <int DT, int NP, bool SWAPPED = false>
__device__ __forceinline__ f32x16 rp_mm(const rp_frag (&a)[NP], const rp_frag (&b)[NP], f32x16 c) {
  if constexpr (NP == 2) {                                   // smallest terms first; the dropped one is below 2^-22 of the product
    c = rp_mm1<DT>(a[!SWAPPED], b[SWAPPED], c);
    c = rp_mm1<DT>(a[SWAPPED], b[!SWAPPED], c);
  }
  return rp_mm1<DT>(a[0], b[0], c);
}
__device__ __forceinline__ f32x16 rp_zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// eight consecutive elements of a row as the type keeps them
template <int DT> struct rp_chunk { uint4 v; };
template <> struct rp_chunk<RP_F32> { f32x4 v[2]; };
template <int DT>
__device__ __forceinline__ rp_chunk<DT> rp_zero_chunk() {
  rp_chunk<DT> c;
  if constexpr (DT == RP_F32) c.v[0] = c.v[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  else c.v = make_uint4(0, 0, 0, 0);
  return c;
}
template <int DT>
__device__ __forceinline__ rp_chunk<DT> rp_load_chunk(const char* p) {
  rp_chunk<DT> c;
  if constexpr (DT == RP_F32) { c.v[0] = reinterpret_cast<const f32x4*>(p)[0]; c.v[1] = reinterpret_cast<const f32x4*>(p)[1]; }
  else c.v = *reinterpret_cast<const uint4*>(p);
  return c;
}
template <int DT>
__device__ __forceinline__ void rp_planes(const rp_chunk<DT>& c, float hs, rp_frag (&out)[rp_type<DT>::NP]) {
  if constexpr (DT == RP_F32) {
    unsigned h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ofb_hsplit_pair(c.v[i >> 1][2 * (i & 1)] * hs, c.v[i >> 1][2 * (i & 1) + 1] * hs, h[i], l[i]);
    out[0] = __builtin_bit_cast(rp_frag, make_uint4(h[0], h[1], h[2], h[3]));
    out[1] = __builtin_bit_cast(rp_frag, make_uint4(l[0], l[1], l[2], l[3]));
  } else {
    out[0] = __builtin_bit_cast(rp_frag, c.v);
  }
}
template <int DT>
__device__ __forceinline__ float rp_chunk_at(const rp_chunk<DT>& c, int i) {
  if constexpr (DT == RP_F32) return c.v[i >> 2][i & 3];
  else if constexpr (DT == RP_BF16) return (float)__builtin_bit_cast(rp_bf16x8, c.v)[i];
  else return (float)__builtin_bit_cast(ofb_f16x8, c.v)[i];
}
__device__ __forceinline__ unsigned rp_pk_bf16(float a, float b) {
  ofb_f32x2 v = {a, b};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, rp_bf16x2));
}
// eight ALREADY SCALED floats as the operand of the second product
template <int DT>
__device__ __forceinline__ void rp_pack8(const float (&x)[8], rp_frag (&out)[rp_type<DT>::NP]) {
  unsigned h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == RP_F32) ofb_hsplit_pair(x[2 * i], x[2 * i + 1], h[i], l[i]);
    else if constexpr (DT == RP_BF16) h[i] = rp_pk_bf16(x[2 * i], x[2 * i + 1]);
    else h[i] = ofb_pk_f16(x[2 * i], x[2 * i + 1]);
  }
  out[0] = __builtin_bit_cast(rp_frag, make_uint4(h[0], h[1], h[2], h[3]));
  if constexpr (DT == RP_F32) out[1] = __builtin_bit_cast(rp_frag, make_uint4(l[0], l[1], l[2], l[3]));
}
// four consecutive elements of an output row
template <int DT>
__device__ __forceinline__ void rp_store4(char* p, float a, float b, float c, float d) {
  if constexpr (DT == RP_F32) *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d};
  else if constexpr (DT == RP_BF16) *reinterpret_cast<uint2*>(p) = make_uint2(rp_pk_bf16(a, b), rp_pk_bf16(c, d));
  else *reinterpret_cast<uint2*>(p) = make_uint2(ofb_pk_f16(a, b), ofb_pk_f16(c, d));
}

// a [rows][DP] tile on its way from memory to LDS: one register image per thread, loaded a tile ahead
template <int DT, int DP, int ROWS>
struct rp_stage {
  using G = rp_geo<DT, DP, ROWS>;
  rp_chunk<DT> c[G::PER];
  __device__ __forceinline__ void load(const char* base, int64_t row_bytes, int row0, int row_end, int d) {
#pragma unroll
    for (int i = 0; i < G::PER; ++i) {
      const int id = threadIdx.x + RP_THREADS * i, row = row0 + id / (DP / 8), ch = (id % (DP / 8)) * 8;
      c[i] = rp_zero_chunk<DT>();
      if (row < row_end && ch < d && (G::CHUNKS % RP_THREADS == 0 || id < G::CHUNKS)) c[i] = rp_load_chunk<DT>(base + (int64_t)row * row_bytes + ch * rp_type<DT>::ES);
    }
  }
  __device__ __forceinline__ void store(char* lds, float hs) const {
#pragma unroll
    for (int i = 0; i < G::PER; ++i) {
      const int id = threadIdx.x + RP_THREADS * i;
      if (G::CHUNKS % RP_THREADS != 0 && id >= G::CHUNKS) continue;
      rp_frag f[G::NP];
      rp_planes<DT>(c[i], hs, f);
#pragma unroll
      for (int p = 0; p < G::NP; ++p) *reinterpret_cast<rp_frag*>(lds + p * G::PLANE + (id / (DP / 8)) * G::PITCH + (id % (DP / 8)) * 16) = f[p];
    }
  }
};

// A operand from an LDS tile, rows along the tile's rows: k-step ks of row0 + (l & 31)
template <int DT, int DP, int ROWS>
__device__ __forceinline__ void rp_rows(const char* lds, int row0, int ks, int lane, rp_frag (&out)[rp_type<DT>::NP]) {
  using G = rp_geo<DT, DP, ROWS>;
#pragma unroll
  for (int p = 0; p < G::NP; ++p) out[p] = *reinterpret_cast<const rp_frag*>(lds + p * G::PLANE + (row0 + (lane & 31)) * G::PITCH + (2 * ks + (lane >> 5)) * 16);
}
// A operand from an LDS tile, rows along the tile's columns (channels 32 ct ..), k-slots = tile rows row0 + 8 (j >> 2) + 4 hh + (j & 3).
// ds_read_b64_tr_b16: in each group of 16 lanes, lane 4 e + q addresses four channels of row e, lane i receives four rows of channel i.
template <int DT, int DP, int ROWS>
__device__ __forceinline__ void rp_cols(const char* lds, int row0, int ct, int lane, rp_frag (&out)[rp_type<DT>::NP]) {
  using G = rp_geo<DT, DP, ROWS>;
  const int off = (row0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * G::PITCH + (32 * ct + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
#pragma unroll
  for (int p = 0; p < G::NP; ++p) {
    const char* q = lds + p * G::PLANE + off;
    const rp_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) rp_s16x4*)(q));
    const rp_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) rp_s16x4*)(q + 8 * G::PITCH));
    out[p] = rp_s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
}

struct rp_scales { int eq, ek, ev, ed, es; };

// exponent of the planes of a tensor whose maximum is b: b 2^e in [2^14, 2^15), as far as the exponents go
__device__ __forceinline__ int rp_exp(float b) {
  if (!(b > 0.f) || !(b < INFINITY)) return 0;
  int ex;
  frexpf(b, &ex);
  return min(15 - ex, RP_EMAX);
}

// The workgroup's tile and head.  Neighbouring tiles of a head share an L2 (its keys or queries are streamed by all of them); causal tiles differ in
// length, so there the longest of all heads come first, and a head stays on one XCD where the number of heads is a multiple of eight.
__device__ __forceinline__ void rp_place(int x, int total, int tiles, bool causal, int& tile, int& bh) {
  if (causal) {
    const int heads = total / tiles;
    tile = x / heads;
    bh = x - tile * heads;
  } else {
    const int id = ofb_xcd_remap(x, total);
    bh = id / tiles;
    tile = id - bh * tiles;
  }
}

// |x| for a maximum.  Infinities and NaN do not count: they pass the planes at any exponent, and the rows that do not meet them keep theirs
__device__ __forceinline__ float rp_size(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }
template <int DT>
__device__ __forceinline__ float rp_size8(const rp_chunk<DT>& c, float top) {
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, rp_size(rp_chunk_at<DT>(c, j)));
  return top;
}
// the maxima of N values over the workgroup, in every thread; red: [4][N]
template <int N>
__device__ __forceinline__ void rp_tops(float (&v)[N], float* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = ofb_wave_max(v[i]);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[(threadIdx.x >> 6) * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = fmaxf(fmaxf(red[i], red[N + i]), fmaxf(red[2 * N + i], red[3 * N + i]));
}
// this thread's share of the maxima over a tensor that are stored for head bh: n of them, step apart from head to head
__device__ __forceinline__ float rp_part(const float* part, int64_t bh, int step, int n) {
  float top = 0.f;
  for (int i = threadIdx.x; i < n; i += RP_THREADS) top = fmaxf(top, part[bh * step + i]);
  return top;
}
// this thread's share of the maxima of one head's first `keys` rows of k and v, eight chunks in flight
template <int DT>
__device__ __forceinline__ void rp_rows_top(const char* k, int64_t k_row, const char* v, int64_t v_row, int keys, int d, float& top_k, float& top_v) {
  const int per = d / 8, groups = RP_THREADS / per, g = threadIdx.x / per, ch = threadIdx.x - g * per;
  top_k = top_v = 0.f;
  if (g >= groups) return;
  k += 8 * ch * rp_type<DT>::ES;
  v += 8 * ch * rp_type<DT>::ES;
  for (int row = g; row < keys; row += 4 * groups) {
    rp_chunk<DT> c[8];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t at = min(row + u * groups, keys - 1);
      c[2 * u] = rp_load_chunk<DT>(k + at * k_row);
      c[2 * u + 1] = rp_load_chunk<DT>(v + at * v_row);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      top_k = rp_size8<DT>(c[2 * u], top_k);
      top_v = rp_size8<DT>(c[2 * u + 1], top_v);
    }
  }
}

// the head's bias by difference, times log2 e, padded by RP_PAD copies of its ends
__device__ __forceinline__ void rp_bias_vector(const ofb_relpos_args& a, int head, float* w) {
  for (int i = threadIdx.x; i < a.width + 2 * RP_PAD; i += RP_THREADS) {
    const int c = min(max(i - RP_PAD, 0), a.width - 1);
    const float t = a.table[(int64_t)a.lut[c] * a.H + head], x = t * 1.44269504088896340736f;
    w[i] = fabsf(t) < INFINITY ? fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f) : x;      // (a finite bias stays one: the type's lowest value as a mask)
  }
}
__device__ __forceinline__ int rp_keys_of(const ofb_relpos_args& a, int b) {
  const int n = a.key_lens ? a.key_lens[b] : a.Nk;
  return min(max(n, 0), a.Nk);
}

// the keys that any query of batch item b sees: what lies behind them may hold anything
__device__ __forceinline__ int rp_seen_of(const ofb_relpos_args& a, int b) {
  const int n = rp_keys_of(a, b);
  return a.causal ? min(n, max(0, a.Nq + a.q_offset)) : n;
}

typedef __attribute__((address_space(3))) const float rp_lds_float;
// the same value in every lane, as a scalar
__device__ __forceinline__ float rp_uniform(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); }
// LDS address of w[RP_PAD]: the entry of difference lo
__device__ __forceinline__ int rp_lds_base(const float* w) { return (int)(uintptr_t)(rp_lds_float*)(w + RP_PAD); }
// the bias at an LDS address, clamped to the head's vector: one instruction (the compiler makes two of min and max), and a read
__device__ __forceinline__ float rp_bias1(int at, int first, int last, int& c) {
  asm("v_med3_i32 %0, %1, %2, %3" : "=v"(c) : "v"(at), "v"(first), "v"(last));
  return *(rp_lds_float*)(uintptr_t)(unsigned)c;
}
__device__ __forceinline__ float rp_bias1(int at, int first, int last) { int c; return rp_bias1(at, first, last, c); }

// register r of an accumulator <-> row of the 32 x 32 tile
__device__ __forceinline__ int rp_row(int r, int hh) { return 8 * (r >> 2) + 4 * hh + (r & 3); }

// the biases of the four pairs whose differences are d0, d0 + step, ... (step +1 or -1): one clamp, one 16-byte read
template <int STEP>
__device__ __forceinline__ int rp_bias4(int w_first, int d0, int width, float (&out)[4]) {
  const int at = w_first + 4 * min(max(STEP > 0 ? d0 : d0 - 3, -RP_PAD), width);
  rp_lds_float* p = (rp_lds_float*)(uintptr_t)(unsigned)at;
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = p[STEP > 0 ? j : 3 - j];
  return at;                                                   // (STEP +1: the first one's LDS address)
}

// ------------------------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------------------------
// A workgroup owns 128 queries of one head (a wave 32 of them, query on the lane), keys stream through two LDS stages.  S^T = K Q^T has
// keys along the registers, so the softmax of a row is register-local but for one exchange between lane halves, and P^T is the B operand of
// O^T = V^T P^T as it stands.
template <int DT, int DP, bool POS, bool SPLIT>
__global__ __launch_bounds__(RP_THREADS, (DP <= 64 ? 3 : DT == RP_F32 ? 1 : 2)) void relpos_fwd_kernel(ofb_relpos_args a) {
  using G = rp_geo<DT, DP, rp_rows_of<DT, DP>(0)>;
  constexpr int NP = G::NP, KB = G::KB, ES = rp_type<DT>::ES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float red[16];
  float* w = reinterpret_cast<float*>(smem);
  int* pk = reinterpret_cast<int*>(smem + ((a.width + 2 * RP_PAD + 3) & ~3) * 4);
  char* tiles = reinterpret_cast<char*>(pk + 2 * KB);
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const int nqt = (a.Nq + RP_TILE - 1) / RP_TILE;
  int qt, bh;
  rp_place(blockIdx.x, gridDim.x, nqt, a.causal, qt, bh);
  if (a.causal) qt = nqt - 1 - qt;                             // the last queries see the most keys
  const int head = bh % a.H, b = bh / a.H;
  const char* qp = (const char*)a.q + (b * a.q_sb + head * a.q_sh) * ES;
  const char* kp = (const char*)a.k + (b * a.k_sb + head * a.k_sh) * ES;
  const char* vp = (const char*)a.v + (b * a.v_sb + head * a.v_sh) * ES;

  int kend = rp_keys_of(a, b);
  const int q_last = min(a.Nq, (qt + 1) * RP_TILE) - 1;
  if (a.causal) kend = min(kend, max(0, q_last + a.q_offset + 1));
  int kb0 = 0, kb1 = (kend + KB - 1) / KB;
  if constexpr (SPLIT) {
    const int per = ((a.Nk + KB - 1) / KB + (int)gridDim.y - 1) / (int)gridDim.y;
    kb0 = min(kb1, per * (int)blockIdx.y);
    kb1 = min(kb1, kb0 + per);
  }

  rp_stage<DT, DP, KB> ks_, vs_;
  int pk_next = 0;
  auto fetch = [&](int kb) {
    ks_.load(kp, a.k_st * ES, kb * KB, kend, a.d);
    vs_.load(vp, a.v_st * ES, kb * KB, kend, a.d);
    if (POS && threadIdx.x < KB) { const int j = kb * KB + threadIdx.x; pk_next = j < kend ? 4 * a.pos_k[j] : 0; }
  };
  if (kb0 < kb1) fetch(kb0);
  rp_bias_vector(a, head, w);
  float hq = 1.f, hk = 1.f, hv = 1.f, c_s = a.scale * 1.44269504088896340736f, c_o = 1.f;
  const int q0 = qt * RP_TILE + wv * 32, qi = q0 + (lane & 31);
  const bool active = q0 < a.Nq, qok = qi < a.Nq;
  const int seen = a.causal ? min(kend, max(0, qi + a.q_offset + 1)) : kend;      // this query sees keys 0 .. seen - 1
  rp_chunk<DT> qc[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int ch = 16 * s + 8 * hh;
    qc[s] = rp_zero_chunk<DT>();
    if (qok && ch < a.d) qc[s] = rp_load_chunk<DT>(qp + (int64_t)qi * a.q_st * ES + ch * ES);
  }
  if constexpr (DT == RP_F32) {
    // exponents of the planes: this tile's for Q, the head's for K and V
    float top[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) top[0] = rp_size8<DT>(qc[s], top[0]);
    if (a.n_bound) {
      top[1] = rp_part(a.bound_k, bh, a.bound_step, a.n_bound);
      top[2] = rp_part(a.bound_v, bh, a.bound_step, a.n_bound);
    } else {
      rp_rows_top<DT>(kp, a.k_st * ES, vp, a.v_st * ES, rp_seen_of(a, b), a.d, top[1], top[2]);
    }
    rp_tops(top, red);
    if (!a.n_bound && a.bound_k && qt == 0 && threadIdx.x == 0) {
      a.bound_k[bh] = top[1];
      a.bound_v[bh] = top[2];
    }
    const int eq = rp_exp(top[0]), ek = rp_exp(top[1]), ev = rp_exp(top[2]);
    hq = ofb_h_pow2(eq); hk = ofb_h_pow2(ek); hv = ofb_h_pow2(ev);
    c_s = __builtin_ldexpf(c_s, -eq - ek);
    c_o = ofb_h_pow2(-ev - RP_PE);                             // P's scale is in it too
  }
  // f32: P's planes hold it times 2^14.  (Not by way of the exponent, where a maximum like -1e9 would swallow it; f16 needs no scale here: P is at
  // most 1 and its row's sum at least 1, what falls below the subnormal step 2^-24 is nothing beside f16's own 2^-11.)
  const float p_sc = DT == RP_F32 ? ofb_h_pow2(RP_PE) : 1.f;

  const int pq = POS ? (qok ? a.pos_q[qi] : 0) : qi + a.q_offset;
  rp_frag qf[DP / 16][NP];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) rp_planes<DT>(qc[s], hq, qf[s]);
  f32x16 O[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) O[t] = rp_zero16();
  float m = -INFINITY, l = 0.f;

  auto commit = [&](int buf) {
    ks_.store(tiles + buf * G::STAGE, hk);
    vs_.store(tiles + buf * G::STAGE + G::TENSOR, hv);
    if (POS && threadIdx.x < KB) pk[buf * KB + threadIdx.x] = pk_next;
  };
  if (kb0 < kb1) commit(0);
  __syncthreads();
  const int lo = a.lo, width = a.width, hi = lo + width - 1, w_first = rp_lds_base(w), w_last = w_first + 4 * (width - 1), pq4 = 4 * (pq + lo) - w_first;
  for (int kb = kb0; kb < kb1; ++kb) {
    const int buf = (kb - kb0) & 1;
    const char* kt_ = tiles + buf * G::STAGE;
    const char* vt_ = kt_ + G::TENSOR;
    if (kb + 1 < kb1) fetch(kb + 1);
    const int j0 = kb * KB;
    if (active && (!a.causal || j0 <= q0 + 31 + a.q_offset)) {
      f32x16 S[KB / 32];
#pragma unroll
      for (int t = 0; t < KB / 32; ++t) {
        S[t] = rp_zero16();
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
          rp_frag kf[NP];
          rp_rows<DT, DP, KB>(kt_, 32 * t, s, lane, kf);
          S[t] = rp_mm<DT, NP>(kf, qf[s], S[t]);
        }
      }
      // scores in log2 units with the bias: s = c_t S + bt, where beyond the table's ends (the whole tile has one bias) S stays as it is
      const int dmax = j0 + KB - 1 - q0 - a.q_offset, dmin = j0 - (q0 + 31) - a.q_offset;
      float bt = 0.f, c_t = 1.f;
      const float wc = rp_uniform(w[RP_PAD + (dmax <= lo ? 0 : width - 1)]);
      // (a large bias, and a scale that is not positive, take the general form)
      const bool one_bias = !POS && (dmax <= lo || dmin >= hi) && fabsf(wc) <= RP_PLAIN && c_s > 0.f;
      if (one_bias) {
        bt = wc;
        c_t = c_s;
      } else if constexpr (POS) {
#pragma unroll
        for (int t = 0; t < KB / 32; ++t)
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            const int4 pj = *reinterpret_cast<const int4*>(&pk[buf * KB + 32 * t + rp_row(r, hh)]);
            S[t][r] = fmaf(S[t][r], c_s, rp_bias1(pj.x - pq4, w_first, w_last));
            S[t][r + 1] = fmaf(S[t][r + 1], c_s, rp_bias1(pj.y - pq4, w_first, w_last));
            S[t][r + 2] = fmaf(S[t][r + 2], c_s, rp_bias1(pj.z - pq4, w_first, w_last));
            S[t][r + 3] = fmaf(S[t][r + 3], c_s, rp_bias1(pj.w - pq4, w_first, w_last));
          }
      } else {
#pragma unroll
        for (int t = 0; t < KB / 32; ++t)
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            float w4[4];
            rp_bias4<1>(w_first, j0 + 32 * t + rp_row(r, hh) - pq - lo, width, w4);
#pragma unroll
            for (int u = 0; u < 4; ++u) S[t][r + u] = fmaf(S[t][r + u], c_s, w4[u]);
          }
      }
      const bool whole = j0 + KB <= kend && (!a.causal || j0 + KB - 1 <= q0 + a.q_offset);
      if (!whole) {
#pragma unroll
        for (int t = 0; t < KB / 32; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (j0 + 32 * t + rp_row(r, hh) >= seen) S[t][r] = -INFINITY;
      }
      float mb = S[0][0];
#pragma unroll
      for (int t = 0; t < KB / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) mb = fmaxf(mb, S[t][r]);
      OFB_XOR_STEP(mb, fmaxf, 32)
      const float m_new = fmaxf(m, fmaf(mb, c_t, bt));
      if (one_bias && __any(fabsf(m_new) > RP_PLAIN)) {        // large scores: rounded, as in the general form
#pragma unroll
        for (int t = 0; t < KB / 32; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) S[t][r] = fmaf(S[t][r], c_t, bt);
        c_t = 1.f;
        bt = 0.f;
      }
      if (__any(m_new > m)) {                                  // the running maximum moves rarely after the first tiles
        const float alpha = m_new > -INFINITY ? __builtin_amdgcn_exp2f(m - m_new) : 1.f;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) O[t] *= alpha;
        m = m_new;
      }
      const float tb = bt - (m > -INFINITY ? m : 0.f);         // a row that has seen nothing yet: exp2(-inf - 0) = 0
#pragma unroll
      for (int t = 0; t < KB / 32; ++t) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float p8[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float p = __builtin_amdgcn_exp2f(fmaf(S[t][8 * s + j], c_t, tb));
            l += p;
            p8[j] = DT == RP_F32 ? p * p_sc : p;
          }
          rp_frag pf[NP];
          rp_pack8<DT>(p8, pf);
#pragma unroll
          for (int ct = 0; ct < DP / 32; ++ct) {
            rp_frag vf[NP];
            rp_cols<DT, DP, KB>(vt_, 32 * t + 16 * s, ct, lane, vf);
            O[ct] = rp_mm<DT, NP>(vf, pf, O[ct]);
          }
        }
      }
    }
    if (kb + 1 < kb1) commit(buf ^ 1);
    __syncthreads();
  }
  OFB_XOR_STEP(l, ofb_add_, 32)
  if (!qok) return;
  const float linv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);             // (a NaN stays one)
  if constexpr (SPLIT) {                                       // the range's own result, joined by relpos_join_kernel
    const int64_t row = ((int64_t)blockIdx.y * a.B * a.H + bh) * a.Nq + qi;
    if (hh == 0) { a.split_ml[2 * row] = m; a.split_ml[2 * row + 1] = l; }
#pragma unroll
    for (int ct = 0; ct < DP / 32; ++ct)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int ch = 32 * ct + rp_row(r, hh);
        if (ch < a.d) *reinterpret_cast<f32x4*>(a.split_o + row * a.d + ch) = f32x4{O[ct][r] * linv * c_o, O[ct][r + 1] * linv * c_o, O[ct][r + 2] * linv * c_o, O[ct][r + 3] * linv * c_o};
      }
  } else {
    if (a.stats && hh == 0) {
      float* st = a.stats + 2 * ((int64_t)bh * a.Nq + qi);
      st[0] = m > -INFINITY ? m : 0.f;
      st[1] = linv;
    }
    char* op = (char*)a.out + (b * a.o_sb + qi * a.o_st + head * a.o_sh) * ES;
    float* o32 = a.out32 ? a.out32 + (((int64_t)b * a.Nq + qi) * a.H + head) * a.d : nullptr;
#pragma unroll
    for (int ct = 0; ct < DP / 32; ++ct)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int ch = 32 * ct + rp_row(r, hh);
        if (ch < a.d) {
          const float x0 = O[ct][r] * linv * c_o, x1 = O[ct][r + 1] * linv * c_o, x2 = O[ct][r + 2] * linv * c_o, x3 = O[ct][r + 3] * linv * c_o;
          rp_store4<DT>(op + ch * ES, x0, x1, x2, x3);
          if (o32) *reinterpret_cast<f32x4*>(o32 + ch) = f32x4{x0, x1, x2, x3};
        }
      }
  }
}

// joins the key ranges of a split forward: one wave per row, lanes along the channels
template <int DT>
__global__ __launch_bounds__(RP_THREADS) void relpos_join_kernel(ofb_relpos_args a, int splits) {
  constexpr int ES = rp_type<DT>::ES;
  const int lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)a.B * a.H * a.Nq, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int qi = (int)(row % a.Nq);
  const int64_t bh = row / a.Nq;
  const int head = (int)(bh % a.H);
  const int64_t b = bh / a.H;
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, a.split_ml[2 * (s * rows + row)]);
  const float mu = m > -INFINITY ? m : 0.f;
  for (int s = 0; s < splits; ++s) l += a.split_ml[2 * (s * rows + row) + 1] * __builtin_amdgcn_exp2f(a.split_ml[2 * (s * rows + row)] - mu);
  const float linv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (a.stats && lane == 0) { a.stats[2 * row] = mu; a.stats[2 * row + 1] = linv; }
  for (int ch = lane * 4; ch < a.d; ch += 256) {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
      const float part = a.split_ml[2 * (s * rows + row) + 1] * __builtin_amdgcn_exp2f(a.split_ml[2 * (s * rows + row)] - mu) * linv;      // the range's share of the row
      o += *reinterpret_cast<const f32x4*>(a.split_o + (s * rows + row) * a.d + ch) * part;
    }
    rp_store4<DT>((char*)a.out + (b * a.o_sb + qi * a.o_st + head * a.o_sh + ch) * ES, o[0], o[1], o[2], o[3]);
    if (a.out32) *reinterpret_cast<f32x4*>(a.out32 + ((b * a.Nq + qi) * a.H + head) * a.d + ch) = o;
  }
}

// ------------------------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------------------------
// top: this thread's share of the maxima of q, k, v and dout (f16: only the last two count)
template <int DT>
__device__ __forceinline__ rp_scales rp_all_scales(float (&top)[4], int d, float* red) {
  rp_scales e = {0, 0, 0, 0, 0};
  if constexpr (DT != RP_BF16) {
    rp_tops(top, red);
    if constexpr (DT == RP_F32) {
      e.eq = rp_exp(top[0]);
      e.ek = rp_exp(top[1]);
      e.ev = rp_exp(top[2]);
      e.ed = rp_exp(top[3]);
    }
    // |dS| <= P (|dP| + |D|) <= 2 d max|dO| max|V| = m 2^ex, m in [0.5, 1): m 2^15 in its scale, as long as that is a power of two that f32 has room for
    // (the factors' exponents apart: their product may leave f32)
    int ev, ed, ec;
    const float m = frexpf(top[2], &ev) * frexpf(top[3], &ed) * frexpf(2.f * d, &ec);
    if (m > 0.f) {
      int ex;
      frexpf(m, &ex);
      e.es = max(RP_EMIN, min(RP_ESMAX, 15 - ex - ev - ed - ec));
    }
  }
  return e;
}

// dQ and D.  The forward's layout: 128 queries a workgroup, the query on the lane; dS^T is the B operand of dQ^T = K^T dS^T from its registers.
// The table's gradient: tiles that lie wholly beyond the first or last difference add up to two numbers, the other pairs go to a histogram by
// difference in LDS, as whole numbers, so that the order of the additions does not matter.  For f32 that happens on the way.  For bf16 and f16 D is
// only known when a row is done (see below): the tiles with pairs between the ends are then visited once more, for S and dP alone.  (A pass of its own
// that summed dS over the batch first, one histogram per pair of tiles, took 170 us beside 98 us of this kernel for the 14 x 14 grid, B 128, 6 x 64
// f32, where this takes 110 us.)
// FEW: see rp_few.
template <int DT, int DP, bool POS, bool FEW>
__global__ __launch_bounds__(RP_THREADS, (DP > 64 && (DT == RP_F32 || FEW) ? 1 : 2)) void relpos_dq_kernel(ofb_relpos_args a) {
  using G = rp_geo<DT, DP, rp_rows_of<DT, DP>(FEW ? 3 : 1)>;
  constexpr int NP = G::NP, KB = G::KB, ES = rp_type<DT>::ES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float red[16];
  const int wpad = (a.width + 2 * RP_PAD + 3) & ~3;
  float* w = reinterpret_cast<float*>(smem);
  unsigned long long* hist = reinterpret_cast<unsigned long long*>(w + wpad);               // [wpad]
  int* pk = reinterpret_cast<int*>(w + 3 * wpad);
  char* tiles = reinterpret_cast<char*>(pk + 2 * KB);
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const int nqt = (a.Nq + RP_TILE - 1) / RP_TILE;
  int qt, bh;
  rp_place(blockIdx.x, gridDim.x, nqt, a.causal, qt, bh);
  if (a.causal) qt = nqt - 1 - qt;                             // the last queries see the most keys
  const int head = bh % a.H, b = bh / a.H;
  const char* qp = (const char*)a.q + (b * a.q_sb + head * a.q_sh) * ES;
  const char* kp = (const char*)a.k + (b * a.k_sb + head * a.k_sh) * ES;
  const char* vp = (const char*)a.v + (b * a.v_sb + head * a.v_sh) * ES;
  const char* dp = (const char*)a.dout + (b * a.do_sb + head * a.do_sh) * ES;
  int kend = rp_keys_of(a, b);
  const int q_last = min(a.Nq, (qt + 1) * RP_TILE) - 1;
  if (a.causal) kend = min(kend, max(0, q_last + a.q_offset + 1));
  const int kb1 = (kend + KB - 1) / KB;
  rp_stage<DT, DP, KB> ks_, vs_;
  int pk_next = 0;
  auto fetch = [&](int kb) {
    ks_.load(kp, a.k_st * ES, kb * KB, kend, a.d);
    vs_.load(vp, a.v_st * ES, kb * KB, kend, a.d);
    if (POS && threadIdx.x < KB) { const int j = kb * KB + threadIdx.x; pk_next = j < kend ? 4 * a.pos_k[j] : 0; }
  };
  if (kb1 > 0) fetch(0);
  rp_bias_vector(a, head, w);
  for (int i = threadIdx.x; i < wpad; i += RP_THREADS) hist[i] = 0ull;
  const int q0 = qt * RP_TILE + wv * 32, qi = q0 + (lane & 31);
  const bool active = q0 < a.Nq, qok = qi < a.Nq;
  const int pq = POS ? (qok ? a.pos_q[qi] : 0) : qi + a.q_offset;
  const int seen = a.causal ? min(kend, max(0, qi + a.q_offset + 1)) : kend;
  rp_chunk<DT> qc[DP / 16], dc[DP / 16];
  float D = 0.f, m = INFINITY, linv = 0.f;                     // (a row behind the last query has P = 0 whatever its biases are)
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int ch = 16 * s + 8 * hh;
    qc[s] = dc[s] = rp_zero_chunk<DT>();
    if (qok && ch < a.d) {
      qc[s] = rp_load_chunk<DT>(qp + (int64_t)qi * a.q_st * ES + ch * ES);
      dc[s] = rp_load_chunk<DT>(dp + (int64_t)qi * a.do_st * ES + ch * ES);
      const float* o32 = a.out32 + (((int64_t)b * a.Nq + qi) * a.H + head) * a.d + ch;
      const f32x4 oa = *reinterpret_cast<const f32x4*>(o32), ob = *reinterpret_cast<const f32x4*>(o32 + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) D = fmaf(rp_chunk_at<DT>(dc[s], j), j < 4 ? oa[j & 3] : ob[j & 3], D);
    }
  }
  // exponents: this tile's for Q, dO and dS, the head's for K and V.  The dK dV kernel reads the tiles' maxima of Q and dO.
  float top[4] = {0.f, 0.f, 0.f, 0.f};
  if constexpr (DT != RP_BF16) {
    // (rows that see nothing count too: the dK dV kernel multiplies them by zeros, so they must stay finite)
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      if constexpr (DT == RP_F32) top[0] = rp_size8<DT>(qc[s], top[0]);
      top[3] = rp_size8<DT>(dc[s], top[3]);
    }
    if constexpr (DT == RP_F32) top[1] = rp_part(a.bound_k, bh, a.bound_step, a.n_bound);
    top[2] = rp_part(a.bound_v, bh, a.bound_step, a.n_bound);
  }
  const rp_scales e = rp_all_scales<DT>(top, a.d, red);
  if (DT != RP_BF16 && threadIdx.x == 0) {
    if constexpr (DT == RP_F32) a.bound_q[(int64_t)bh * nqt + qt] = top[0];
    a.bound_do[(int64_t)bh * nqt + qt] = top[3];
  }
  const float hq = ofb_h_pow2(e.eq), hk = ofb_h_pow2(e.ek), hv = ofb_h_pow2(e.ev), hd = ofb_h_pow2(e.ed);
  const float c_s = __builtin_ldexpf(a.scale * 1.44269504088896340736f, -e.eq - e.ek);
  const int ek_ = e.es - e.ed - e.ev;                          // dP's accumulators times 2^ek_ are in dS's scale
  rp_frag qf[DP / 16][NP], df[DP / 16][NP];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    rp_planes<DT>(qc[s], hq, qf[s]);
    rp_planes<DT>(dc[s], hd, df[s]);
  }
  OFB_XOR_STEP(D, ofb_add_, 32)
  if (qok) {
    const int64_t row = (int64_t)bh * a.Nq + qi;
    m = a.stats[2 * row];
    linv = a.stats[2 * row + 1];
  }
  // Inside the loop P lacks its factor 1 / sum, a constant of the lane that the row's results take at the end, and is held times kk.  (Neither goes
  // into the exponent: a maximum like -1e9 would swallow it.)
  const float kk = DT == RP_BF16 ? 1.f : ofb_h_pow2(max(-126, min(126, ek_))), nD = -__builtin_ldexpf(D, e.ed + e.ev);
  f32x16 dQ[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) dQ[t] = rp_zero16();
  float sat_lo = 0.f, sat_hi = 0.f, pat_lo = 0.f, pat_hi = 0.f, left = 0.f;
  auto commit = [&](int buf) {
    ks_.store(tiles + buf * G::STAGE, hk);
    vs_.store(tiles + buf * G::STAGE + G::TENSOR, hv);
    if (POS && threadIdx.x < KB) pk[buf * KB + threadIdx.x] = pk_next;
  };
  if (kb1 > 0) commit(0);
  const bool plain = !__syncthreads_or(qok && fabsf(m) > RP_PLAIN);        // (of the workgroup: its waves share the second visit's tiles)
  const int lo = a.lo, width = a.width, hi = lo + width - 1, w_first = rp_lds_base(w), w_last = w_first + 4 * (width - 1), pq4 = 4 * (pq + lo) - w_first;
  // S and dP - D (in dP's scale) of 32 keys
  auto products = [&](const char* kt_, const char* vt_, int t0, float nd, f32x16& S, f32x16& dP) {
    S = rp_zero16();
#pragma unroll
    for (int r = 0; r < 16; ++r) dP[r] = nd;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      rp_frag kf[NP], vf[NP];
      rp_rows<DT, DP, KB>(kt_, 32 * t0, s, lane, kf);
      rp_rows<DT, DP, KB>(vt_, 32 * t0, s, lane, vf);
      S = rp_mm<DT, NP>(kf, qf[s], S);
      dP = rp_mm<DT, NP>(vf, df[s], dP);
    }
  };
  // ds: dS over 1 / sum, in units of 1 / k, k = the power of two that makes it the second product's operand (dP's own scale is in it too).
  // at: the LDS addresses of the pairs' biases.
  auto general = [&](f32x16& S, f32x16& dP, int buf, int t0, int j0, bool whole, float (&ds)[16], int (&at)[16]) {
    float t[16];
    if constexpr (POS) {
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int4 pj = *reinterpret_cast<const int4*>(&pk[buf * KB + 32 * t0 + rp_row(r, hh)]);
        t[r] = rp_bias1(pj.x - pq4, w_first, w_last, at[r]);
        t[r + 1] = rp_bias1(pj.y - pq4, w_first, w_last, at[r + 1]);
        t[r + 2] = rp_bias1(pj.z - pq4, w_first, w_last, at[r + 2]);
        t[r + 3] = rp_bias1(pj.w - pq4, w_first, w_last, at[r + 3]);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        float w4[4];
        at[r] = rp_bias4<1>(w_first, j0 + rp_row(r, hh) - pq - lo, width, w4);
#pragma unroll
        for (int u = 0; u < 4; ++u) { t[r + u] = w4[u]; at[r + u] = at[r] + 4 * u; }
      }
    }
    if (!whole) {                                              // keys this query does not see: P = 0, whatever S and dP are there
      asm volatile("");
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (j0 + rp_row(r, hh) >= seen) { t[r] = -INFINITY; S[r] = dP[r] = 0.f; }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      ds[r] = __builtin_amdgcn_exp2f(fmaf(S[r], c_s, t[r]) - m) * kk * dP[r];
    }
  };
  // adds the pairs to their bins as whole numbers of 2^-32 / mul: high word floor(mul ds), low word the rest
  auto bins = [&](const float (&ds)[16], const int (&at)[16], float mul) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float y = ds[r] * mul;
      const unsigned long long v = ((unsigned long long)(unsigned)(int)floorf(y) << 32) | (unsigned)(__builtin_amdgcn_fractf(y) * 4294967296.f);
      atomicAdd(reinterpret_cast<unsigned long long*>(reinterpret_cast<char*>(hist) + 2 * (at[r] - w_first + 4 * RP_PAD)), v);
    }
  };
  auto visible = [&](int j0) { return active && j0 < kend && !(a.causal && j0 > q0 + 31 + a.q_offset); };
  auto is_whole = [&](int j0, int n, int first) { return j0 + n <= kend && (!a.causal || j0 + n - 1 <= first + a.q_offset); };
  // the whole tile of keys j0 .. j0 + n - 1 and queries first .. last lies beyond an end: -1, 1 or 0
  // (large biases and scores take the general form, as in the forward)
  const float w_lo = rp_uniform(w[RP_PAD]), w_hi = rp_uniform(w[RP_PAD + width - 1]);
  const int below = plain && fabsf(w_lo) <= RP_PLAIN ? lo + a.q_offset : -0x7fffffff, above = plain && fabsf(w_hi) <= RP_PLAIN ? hi + a.q_offset : 0x7fffffff;
  auto beyond = [&](int j0, int n, int first, int last) { return POS ? 0 : j0 + n - 1 - first <= below ? -1 : j0 - last >= above ? 1 : 0; };
  float most = 0.f;                                            // the largest |ds| that goes to a bin
  for (int kb = 0; kb < kb1; ++kb) {
    const int buf = kb & 1;
    const char* kt_ = tiles + buf * G::STAGE;
    const char* vt_ = kt_ + G::TENSOR;
    if (kb + 1 < kb1) fetch(kb + 1);
#pragma unroll 2
    for (int t0 = 0; t0 < KB / 32; ++t0) {
      const int j0 = kb * KB + 32 * t0;
      if (!visible(j0)) continue;
      f32x16 S, dP;
      products(kt_, vt_, t0, nD, S, dP);
      const bool whole = is_whole(j0, 32, q0);
      const int side = beyond(j0, 32, q0, q0 + 31);
      float ds[16], sum = 0.f;
      if (!POS && whole && side) {
        const float tb = (side < 0 ? w_lo : w_hi) - m;
        float psum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = __builtin_amdgcn_exp2f(fmaf(S[r], c_s, tb)) * kk;
          ds[r] = p * dP[r];
          sum += ds[r];
          psum += p;
        }
        if (side < 0) { sat_lo += sum; pat_lo += psum; } else { sat_hi += sum; pat_hi += psum; }
      } else {
        int at[16];
        general(S, dP, buf, t0, j0, whole, ds, at);
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += ds[r];
        if constexpr (DT == RP_F32) {                          // |ds| < 2^15, and a row's |ds| sum to less than that: 128 rows stay below 2^60
          if (a.dtable) { asm volatile(""); bins(ds, at, 64.f * linv); }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(ds[r]));
        }
      }
      left += sum;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float x8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x8[j] = ds[8 * s + j];
        rp_frag xf[NP];
        rp_pack8<DT>(x8, xf);
#pragma unroll
        for (int ct = 0; ct < DP / 32; ++ct) {
          rp_frag kf[NP];
          rp_cols<DT, DP, KB>(kt_, 32 * t0 + 16 * s, ct, lane, kf);
          dQ[ct] = rp_mm<DT, NP>(kf, xf, dQ[ct]);
        }
      }
    }
    if (kb + 1 < kb1) commit(buf ^ 1);
    __syncthreads();
  }
  const float c_dq = a.scale * linv;
  const int e_dq = -e.es - e.ek;                               // (apart from the factor: the two together may leave f32)
  if (qok) {
    char* op = (char*)a.dq + (b * a.dq_sb + qi * a.dq_st + head * a.dq_sh) * ES;
#pragma unroll
    for (int ct = 0; ct < DP / 32; ++ct)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int ch = 32 * ct + rp_row(r, hh);
        if (ch < a.d) rp_store4<DT>(op + ch * ES, __builtin_ldexpf(dQ[ct][r] * c_dq, e_dq), __builtin_ldexpf(dQ[ct][r + 1] * c_dq, e_dq),
                                    __builtin_ldexpf(dQ[ct][r + 2] * c_dq, e_dq), __builtin_ldexpf(dQ[ct][r + 3] * c_dq, e_dq));
      }
  }
  // D came from an output whose P was rounded for the product.  A row of dS sums to zero, so what this row's sum is off by is D's error: the
  // kernels that follow read D without it, and the sums above lose it times their share of P.  (The table's gradient is f32 and sums whole rows'
  // parts, where an error that a row's terms share does not average out: without this it was 1e-3 off for bf16.)
  OFB_XOR_STEP(left, ofb_add_, 32)
  left *= linv;
  if (qok && hh == 0) a.delta[(int64_t)bh * a.Nq + qi] = D + __builtin_ldexpf(left, -e.es);
  if (!a.dtable) return;
  if (a.sat) {
    const float k = __builtin_ldexpf(left, -ek_);              // (P is held times 2^ek_ and without 1 / sum)
    sat_lo = ofb_wave_sum((sat_lo - k * pat_lo) * linv);
    sat_hi = ofb_wave_sum((sat_hi - k * pat_hi) * linv);
    if (lane == 0) {
      const int64_t n = (int64_t)a.B * nqt * 4, at = ((int64_t)b * nqt + qt) * 4 + wv;
      a.sat[(2 * (int64_t)head) * n + at] = __builtin_ldexpf(sat_lo, -e.es);
      a.sat[(2 * (int64_t)head + 1) * n + at] = __builtin_ldexpf(sat_hi, -e.es);
    }
  }
  const bool bad = __syncthreads_or(!(fabsf(left) < 3.0e38f));             // (the conversions drop NaN and infinities)
  int unit = 38;
  if constexpr (DT != RP_F32) {
    // once more over the tiles with pairs between the ends, with the D that is known now; bins of 2^-unit, such that all pairs of the
    // workgroup could be as large as the largest
    most = ofb_wave_max(most * linv + fabsf(left));
    if (lane == 0) red[wv] = most;
    __syncthreads();
    most = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    int ex = 0;
    if (most > 0.f) frexpf(most, &ex);
    unit = 62 - max(ex, -60) - (7 + 32 - __clz(a.Nk));
    const float mul = __builtin_ldexpf(linv, unit - 32), nd = nD - __builtin_ldexpf(left, e.ed + e.ev - e.es);
    // (to the end of the last wave's 32 rows, as in the waves' own tests: what a wave has not summed as a whole must be visited)
    auto next = [&](int kb) {
      while (kb < kb1 && is_whole(kb * KB, KB, qt * RP_TILE) && beyond(kb * KB, KB, qt * RP_TILE, q_last | 31)) ++kb;
      return kb;
    };
    int kb = bad ? kb1 : next(0), buf = 0;
    if (kb < kb1) { fetch(kb); commit(0); }
    __syncthreads();
    while (kb < kb1) {
      const char* kt_ = tiles + buf * G::STAGE;
      const int after = next(kb + 1);
      if (after < kb1) fetch(after);
      for (int t0 = 0; t0 < KB / 32; ++t0) {
        const int j0 = kb * KB + 32 * t0;
        const bool whole = is_whole(j0, 32, q0);
        if (!visible(j0) || (whole && beyond(j0, 32, q0, q0 + 31))) continue;
        f32x16 S, dP;
        float ds[16];
        int at[16];
        products(kt_, kt_ + G::TENSOR, t0, nd, S, dP);
        general(S, dP, buf, t0, j0, whole, ds, at);
        bins(ds, at, mul);
      }
      if (after < kb1) commit(buf ^ 1);
      __syncthreads();
      kb = after;
      buf ^= 1;
    }
  }
  const int64_t rows = (int64_t)a.B * nqt, at = (int64_t)b * nqt + qt;
  for (int i = threadIdx.x; i < width; i += RP_THREADS) {
    long long v = (long long)hist[i + RP_PAD];
    if (i == 0)
      for (int u = 0; u < RP_PAD; ++u) v += (long long)hist[u];
    if (i == width - 1)
      for (int u = 0; u < RP_PAD; ++u) v += (long long)hist[width + RP_PAD + u];
    a.partial[((int64_t)head * width + i) * rows + at] = bad ? __builtin_nanf("") : (float)__builtin_ldexp((double)v, -unit - e.es);
  }
}

// a query tile's row statistics for LDS: the maximum, 1 / sum times the operand's scale 2^pe, -D in dP's scale 2^de; a row without keys has 1 / sum 0, one
// behind the last query a maximum of infinity: P = 0
template <int KB, bool POS>
__device__ __forceinline__ void rp_row_stats(const ofb_relpos_args& a, int64_t bh, int row0, int pe, int de, f32x4& v, int& pos) {
  const int i = row0 + threadIdx.x;
  v = f32x4{INFINITY, 0.f, 0.f, 0.f};                          // (a maximum of 0 would leave exp2 of a large bias there: infinity times 0)
  pos = 0;
  if (threadIdx.x < KB && i < a.Nq) {
    const int64_t row = bh * a.Nq + i;
    v[0] = a.stats[2 * row];
    v[1] = __builtin_ldexpf(a.stats[2 * row + 1], pe);
    v[2] = -__builtin_ldexpf(a.delta[row], de);
    pos = POS ? 4 * a.pos_q[i] : i + a.q_offset;
  }
}

// P and dS of a 32 x 32 tile, rows = queries i0 .. (LDS tiles qt_ and dt_ at row tr), the wave's key on the lane.  st: row statistics m, l, -D of
// the tile's queries, -D in dP's scale.  P = exp2(s - m) l comes out times the scale that is in l, dS = P (dP - D) times that and dP's scale.  (1 / sum stays
// apart: its logarithm does not survive beside a maximum like -1e9.)
template <int DT, int DP, int ROWS, bool POS>
__device__ __forceinline__ void rp_tile_ds(const ofb_relpos_args& a, const char* qt_, const char* dt_, int tr, const rp_frag (&kf)[DP / 16][rp_type<DT>::NP],
                                           const rp_frag (&vf)[DP / 16][rp_type<DT>::NP], const float* st, const int* ps, const float* w, int i0, int j0,
                                           int kj, int pkj, bool kok, bool kwhole, float c_s, float (&P)[16], float (&dS)[16]) {
  using G = rp_geo<DT, DP, ROWS>;
  constexpr int NP = G::NP, KB = G::KB;
  const int lane = threadIdx.x & 63, hh = lane >> 5, lo = a.lo, width = a.width, hi = lo + width - 1, w_first = rp_lds_base(w),
            w_last = w_first + 4 * (width - 1), pk4 = 4 * (pkj - lo) + w_first;
  f32x16 S = rp_zero16(), dP;
#pragma unroll
  for (int r = 0; r < 16; r += 4) {
    const f32x4 d4 = *reinterpret_cast<const f32x4*>(&st[2 * KB + tr + rp_row(r, hh)]);
#pragma unroll
    for (int u = 0; u < 4; ++u) dP[r + u] = d4[u];
  }
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    rp_frag qa[NP], da[NP];
    rp_rows<DT, DP, KB>(qt_, tr, s, lane, qa);
    rp_rows<DT, DP, KB>(dt_, tr, s, lane, da);
    S = rp_mm<DT, NP, true>(qa, kf[s], S);                      // the forward's S: its weights are 1 at most whatever the scores' size is
    dP = rp_mm<DT, NP, true>(da, vf[s], dP);
  }
  const int dmax = j0 + 31 - i0 - a.q_offset, dmin = j0 - (i0 + 31) - a.q_offset;
  const bool cut = a.causal && j0 + 31 > i0 + a.q_offset;
  float t[16];
  if (!POS && (dmax <= lo || dmin >= hi)) {
    const float wc = w[RP_PAD + (dmax <= lo ? 0 : width - 1)];
#pragma unroll
    for (int r = 0; r < 16; ++r) t[r] = wc;
  } else if constexpr (POS) {
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int4 pi = *reinterpret_cast<const int4*>(&ps[tr + rp_row(r, hh)]);
      t[r] = rp_bias1(pk4 - pi.x, w_first, w_last);
      t[r + 1] = rp_bias1(pk4 - pi.y, w_first, w_last);
      t[r + 2] = rp_bias1(pk4 - pi.z, w_first, w_last);
      t[r + 3] = rp_bias1(pk4 - pi.w, w_first, w_last);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      float w4[4];
      rp_bias4<-1>(w_first, kj - (i0 + rp_row(r, hh) + a.q_offset) - lo, width, w4);
#pragma unroll
      for (int u = 0; u < 4; ++u) t[r + u] = w4[u];
    }
  }
  if (!kwhole || cut) {                                        // queries that do not see this key: P = 0, whatever S and dP are there
    asm volatile("");
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (!kok || (cut && kj > i0 + rp_row(r, hh) + a.q_offset)) { t[r] = -INFINITY; S[r] = dP[r] = 0.f; }
  }
#pragma unroll
  for (int r = 0; r < 16; r += 4) {
    const int rr = rp_row(r, hh);
    const f32x4 m4 = *reinterpret_cast<const f32x4*>(&st[tr + rr]), l4 = *reinterpret_cast<const f32x4*>(&st[KB + tr + rr]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      P[r + u] = __builtin_amdgcn_exp2f(fmaf(S[r + u], c_s, t[r + u]) - m4[u]) * l4[u];
      dS[r + u] = P[r + u] * dP[r + u];
    }
  }
}

// dK and dV: a workgroup owns 128 keys of one head (a wave 32, key on the lane, K and V in registers), queries stream through LDS.
// S = Q K^T and dP = dO V^T have queries along the registers: P and dS are the B operands of dV^T = dO^T P and dK^T = Q^T dS.
template <int DT, int DP, bool POS>
__global__ __launch_bounds__(RP_THREADS, (DP <= 64 ? 2 : 1)) void relpos_dkv_kernel(ofb_relpos_args a) {
  using G = rp_geo<DT, DP, rp_rows_of<DT, DP>(2)>;
  constexpr int NP = G::NP, KB = G::KB, ES = rp_type<DT>::ES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float red[16];
  float* w = reinterpret_cast<float*>(smem);
  float* st = reinterpret_cast<float*>(smem + ((a.width + 2 * RP_PAD + 3) & ~3) * 4);      // [2][3][KB]
  int* ps = reinterpret_cast<int*>(st + 6 * KB);                                            // [2][KB]
  char* tiles = reinterpret_cast<char*>(ps + 2 * KB);
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const int nkt = (a.Nk + RP_TILE - 1) / RP_TILE;
  int kt, bh;
  rp_place(blockIdx.x, gridDim.x, nkt, a.causal, kt, bh);
  const int head = bh % a.H, b = bh / a.H;
  const char* qp = (const char*)a.q + (b * a.q_sb + head * a.q_sh) * ES;
  const char* kp = (const char*)a.k + (b * a.k_sb + head * a.k_sh) * ES;
  const char* vp = (const char*)a.v + (b * a.v_sb + head * a.v_sh) * ES;
  const char* dp = (const char*)a.dout + (b * a.do_sb + head * a.do_sh) * ES;
  const int kend = rp_seen_of(a, b), j_first = kt * RP_TILE;
  int qb0 = 0, qb1 = (a.Nq + KB - 1) / KB;
  if (a.causal) qb0 = min(qb1, max(0, j_first - a.q_offset) / KB);
  if (j_first >= kend) qb0 = qb1;                              // nobody sees these keys: their gradients are zeros
  float top[4] = {0.f, 0.f, 0.f, 0.f};
  if constexpr (DT != RP_BF16) {
    const int nqt = (a.Nq + RP_TILE - 1) / RP_TILE;
    if constexpr (DT == RP_F32) {
      top[0] = rp_part(a.bound_q, bh, nqt, nqt);
      top[1] = rp_part(a.bound_k, bh, a.bound_step, a.n_bound);
    }
    top[2] = rp_part(a.bound_v, bh, a.bound_step, a.n_bound);
    top[3] = rp_part(a.bound_do, bh, nqt, nqt);
  }
  const rp_scales e = rp_all_scales<DT>(top, a.d, red);
  rp_stage<DT, DP, KB> qs_, ds_;
  f32x4 st_next;
  int ps_next;
  auto fetch = [&](int qb) {
    qs_.load(qp, a.q_st * ES, qb * KB, a.Nq, a.d);
    ds_.load(dp, a.do_st * ES, qb * KB, a.Nq, a.d);
    rp_row_stats<KB, POS>(a, bh, qb * KB, DT == RP_BF16 ? 0 : RP_PE, e.ed + e.ev, st_next, ps_next);
  };
  rp_bias_vector(a, head, w);
  if (qb0 < qb1) fetch(qb0);
  const float hq = ofb_h_pow2(e.eq), hk = ofb_h_pow2(e.ek), hv = ofb_h_pow2(e.ev), hd = ofb_h_pow2(e.ed);
  const float c_s = __builtin_ldexpf(a.scale * 1.44269504088896340736f, -e.eq - e.ek);
  const float c_x = DT == RP_BF16 ? 1.f : ofb_h_pow2(e.es - e.ed - e.ev - RP_PE);      // dS from rp_tile_ds to the operand's scale
  const int e_dk = -e.es - e.eq;
  const float c_dv = DT == RP_BF16 ? 1.f : ofb_h_pow2(-RP_PE - e.ed);

  const int j0 = j_first + wv * 32, kj = j0 + (lane & 31);
  const bool active = j0 < kend, kok = kj < kend;
  const int pkj = POS ? (kok ? a.pos_k[kj] : 0) : kj;
  rp_frag kf[DP / 16][NP], vf[DP / 16][NP];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int ch = 16 * s + 8 * hh;
    rp_chunk<DT> c = rp_zero_chunk<DT>(), g = rp_zero_chunk<DT>();
    if (kok && ch < a.d) {
      c = rp_load_chunk<DT>(kp + (int64_t)kj * a.k_st * ES + ch * ES);
      g = rp_load_chunk<DT>(vp + (int64_t)kj * a.v_st * ES + ch * ES);
    }
    rp_planes<DT>(c, hk, kf[s]);
    rp_planes<DT>(g, hv, vf[s]);
  }
  f32x16 dK[DP / 32], dV[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) dK[t] = dV[t] = rp_zero16();
  auto commit = [&](int buf) {
    qs_.store(tiles + buf * G::STAGE, hq);
    ds_.store(tiles + buf * G::STAGE + G::TENSOR, hd);
    if (threadIdx.x < KB) {
#pragma unroll
      for (int u = 0; u < 3; ++u) st[(buf * 3 + u) * KB + threadIdx.x] = st_next[u];
      ps[buf * KB + threadIdx.x] = ps_next;
    }
  };
  if (qb0 < qb1) commit(0);
  __syncthreads();
  for (int qb = qb0; qb < qb1; ++qb) {
    const int buf = (qb - qb0) & 1;
    const char* qt_ = tiles + buf * G::STAGE;
    const char* dt_ = qt_ + G::TENSOR;
    if (qb + 1 < qb1) fetch(qb + 1);
#pragma unroll 2
    for (int t = 0; t < KB / 32; ++t) {
      const int i0 = qb * KB + 32 * t;
      if (!active || i0 >= a.Nq || (a.causal && j0 > i0 + 31 + a.q_offset)) continue;
      float P[16], dS[16];
      rp_tile_ds<DT, DP, KB, POS>(a, qt_, dt_, 32 * t, kf, vf, st + buf * 3 * KB, ps + buf * KB, w, i0, j0, kj, pkj, kok, j0 + 32 <= kend, c_s, P, dS);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float p8[8], x8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { p8[j] = P[8 * s + j]; x8[j] = DT == RP_BF16 ? dS[8 * s + j] : dS[8 * s + j] * c_x; }
        rp_frag pf[NP], xf[NP];
        rp_pack8<DT>(p8, pf);
        rp_pack8<DT>(x8, xf);
#pragma unroll
        for (int ct = 0; ct < DP / 32; ++ct) {
          rp_frag df[NP], qf[NP];
          rp_cols<DT, DP, KB>(dt_, 32 * t + 16 * s, ct, lane, df);
          rp_cols<DT, DP, KB>(qt_, 32 * t + 16 * s, ct, lane, qf);
          dV[ct] = rp_mm<DT, NP>(df, pf, dV[ct]);
          dK[ct] = rp_mm<DT, NP>(qf, xf, dK[ct]);
        }
      }
    }
    if (qb + 1 < qb1) commit(buf ^ 1);
    __syncthreads();
  }
  if (kj >= a.Nk) return;
  char* okp = (char*)a.dk + (b * a.dk_sb + kj * a.dk_st + head * a.dk_sh) * ES;
  char* ovp = (char*)a.dv + (b * a.dv_sb + kj * a.dv_st + head * a.dv_sh) * ES;
#pragma unroll
  for (int ct = 0; ct < DP / 32; ++ct)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int ch = 32 * ct + rp_row(r, hh);
      if (ch < a.d) {
        rp_store4<DT>(okp + ch * ES, __builtin_ldexpf(dK[ct][r] * a.scale, e_dk), __builtin_ldexpf(dK[ct][r + 1] * a.scale, e_dk),
                      __builtin_ldexpf(dK[ct][r + 2] * a.scale, e_dk), __builtin_ldexpf(dK[ct][r + 3] * a.scale, e_dk));
        rp_store4<DT>(ovp + ch * ES, dV[ct][r] * c_dv, dV[ct][r + 1] * c_dv, dV[ct][r + 2] * c_dv, dV[ct][r + 3] * c_dv);
      }
    }
}

// table gradient: one workgroup per (bucket, head) adds up the differences of its bucket over all workgroups of the dQ kernel, in a fixed order and in
// 64 bits.  (difference, workgroup) pairs are dealt out together: buckets hold from one difference to dozens.
__global__ __launch_bounds__(RP_THREADS) void relpos_table_kernel(ofb_relpos_args a, int64_t rows, int64_t nsat) {
  __shared__ double red[4];
  const int c = blockIdx.x / a.H, head = blockIdx.x % a.H, e0 = a.bucket_start[c];
  const int64_t items = (a.bucket_start[c + 1] - e0) * rows;
  double sum = 0.0;
#pragma unroll 4
  for (int64_t it = threadIdx.x; it < items; it += RP_THREADS) {
    const int64_t e = it / rows;
    sum += (double)a.partial[((int64_t)head * a.width + a.bucket_order[e0 + e]) * rows + (it - e * rows)];
  }
  if (nsat > 0) {                                              // the sums beyond the ends belong to the ends' buckets
    for (int side = 0; side < 2; ++side) {
      if (a.lut[side ? a.width - 1 : 0] != c) continue;
      const float* p = a.sat + (2 * (int64_t)head + side) * nsat;
      for (int64_t r = threadIdx.x; r < nsat; r += RP_THREADS) sum += (double)p[r];
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.dtable[(int64_t)c * a.H + head] = (float)(red[0] + red[1] + red[2] + red[3]);
}

// partial maxima of |x| of k and / or v (blockIdx.y), over the keys that can be seen: what lies behind them may hold anything
template <int DT>
__global__ __launch_bounds__(RP_THREADS) void relpos_amax_kernel(ofb_relpos_args a, int first) {
  constexpr int ES = rp_type<DT>::ES;
  __shared__ float red[4];
  const bool is_k = first + blockIdx.y == 0;
  const char* x = (const char*)(is_k ? a.k : a.v);
  const int64_t sb = is_k ? a.k_sb : a.v_sb, st = is_k ? a.k_st : a.v_st, sh = is_k ? a.k_sh : a.v_sh;
  const int per = a.H * (a.d / 8);                             // chunks of a token
  const int tokens = a.Nk;
  float v = 0.f;
  const int64_t rows = (int64_t)a.B * tokens;
  // a group of threads per token (`per` chunks each), four tokens' loads in flight
  const int group = min(per, RP_THREADS), groups = RP_THREADS / group, g = threadIdx.x / group, t0 = threadIdx.x % group;
  const int64_t step = (int64_t)gridDim.x * groups;
  if (g < groups) {
    for (int64_t row = (int64_t)blockIdx.x * groups + g; row < rows; row += 4 * step) {
      const char* p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t at = row + u * step;
        const int b = (int)(at / tokens), i = (int)(at - (int64_t)b * tokens);
        p[u] = nullptr;
        if (at >= rows) continue;
        if (i < rp_seen_of(a, b)) p[u] = x + (b * sb + (int64_t)i * st) * ES;
      }
      for (int c = t0; c < per; c += group) {
        const int64_t off = ((c / (a.d / 8)) * sh + (c % (a.d / 8)) * 8) * ES;
        rp_chunk<DT> q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          q[u] = rp_zero_chunk<DT>();
          if (p[u]) q[u] = rp_load_chunk<DT>(p[u] + off);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) v = rp_size8<DT>(q[u], v);
      }
    }
  }
  float top[1] = {v};
  rp_tops(top, red);
  if (threadIdx.x == 0) (is_k ? a.bound_k : a.bound_v)[blockIdx.x] = top[0];
}

template <int DT, int DP, int KERNEL> int rp_lds(const ofb_relpos_args& a) {
  using G = rp_geo<DT, DP, rp_rows_of<DT, DP>(KERNEL)>;
  const int w = ((a.width + 2 * RP_PAD + 3) & ~3) * 4;
  return w * (KERNEL & 1 ? 3 : 1) + (KERNEL == 2 ? 8 : 2) * G::KB * 4 + 2 * G::STAGE;
}

template <typename F> int rp_allow(F* f, int bytes) {
  return bytes <= 65536 ? 0 : (int)hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
#define RP_LAUNCH(kernel, grid, lds, stream, ...)                                                                    \
  do {                                                                                                               \
    if (const int rc_ = rp_allow(kernel, lds)) return rc_;                                                           \
    hipLaunchKernelGGL(kernel, grid, dim3(RP_THREADS), lds, stream, __VA_ARGS__);                                    \
  } while (0)

int rp_kb(const ofb_relpos_args& a) { return a.dtype == RP_F32 ? rp_rows_of<RP_F32, 64>(0) : a.d <= 64 ? rp_rows_of<RP_BF16, 64>(0) : rp_rows_of<RP_BF16, 128>(0); }
// workgroups per head that leave a part of the table's gradient
int64_t rp_table_rows(const ofb_relpos_args& a) { return (int64_t)a.B * ((a.Nq + RP_TILE - 1) / RP_TILE); }

// key ranges of the forward, where the query tiles leave the chip idle: a range costs a partial output, written and read again, for every query.  Up to 32
// queries (one wave; the others stage) that is nothing beside the keys.  For more, only whole multiples are worth it: 4 x 1025 causal queries, 8 heads of
// 128 f16, are 288 workgroups and take 40 + 27 us in four ranges, 54 us in one.
int rp_splits(const ofb_relpos_args& a) {
  const int64_t wgs = (int64_t)a.B * a.H * ((a.Nq + RP_TILE - 1) / RP_TILE), nkb = (a.Nk + rp_kb(a) - 1) / rp_kb(a);
  const int64_t want = a.Nq <= 32 ? (1024 + wgs - 1) / wgs : 512 / wgs, most = nkb / 4;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

// f32: a workgroup of the forward finds its head's maxima of K and V by itself where that is little to read once more
bool rp_own_bounds(const ofb_relpos_args& a) { return a.dtype == RP_F32 && a.Nk <= RP_OWN && rp_splits(a) == 1; }

int rp_check(const ofb_relpos_args* a) {
  if (!a || !a->q || !a->k || !a->v || !a->table || !a->lut) return OFB_EINVAL;
  if (a->B < 1 || a->H < 1 || a->Nq < 1 || a->Nk < 1 || a->d < 8 || a->d % 8 || a->dtype < 0 || a->dtype > 2) return OFB_EINVAL;
  if (a->width < 1 || a->n_buckets < 1 || (!a->pos_q) != (!a->pos_k) || (a->pos_q && a->causal)) return OFB_EINVAL;
  if (a->d > 128 || a->width > RP_WMAX || a->n_buckets > (1 << 20) || a->Nq > (1 << 26) || a->Nk > (1 << 26)) return OFB_ELIMIT;
  if (a->q_offset > (1 << 26) || a->q_offset < -(1 << 26) || a->lo > (1 << 26) || a->lo < -(1 << 26)) return OFB_ELIMIT;
  const int64_t tiles = (int64_t)a->B * a->H * (((int64_t)(a->Nq > a->Nk ? a->Nq : a->Nk) + RP_TILE - 1) / RP_TILE);
  if (tiles >= (1 << 24)) return OFB_ELIMIT;                   // threads of a launch count in 32 bits
  const int64_t unit = a->dtype == RP_F32 ? 4 : 8;             // 16-byte loads
  if (!ofb_aligned16(a->q) || !ofb_aligned16(a->k) || !ofb_aligned16(a->v)) return OFB_EINVAL;
  for (int64_t s : {a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh, a->v_sb, a->v_st, a->v_sh})
    if (s % unit || s < 0) return OFB_EINVAL;
  if (a->n_bound < 0 || a->n_bound > RP_NBOUND || a->bound_step < 0 || a->bound_step > RP_NBOUND) return OFB_EINVAL;
  return OFB_OK;
}

template <int DT, int DP, bool POS> int rp_forward_of(const ofb_relpos_args& a, hipStream_t s) {
  const int64_t wgs = (int64_t)a.B * a.H * ((a.Nq + RP_TILE - 1) / RP_TILE);
  const int lds = rp_lds<DT, DP, 0>(a), splits = rp_splits(a);
  if (splits > 1) {
    if (!a.split_o || !a.split_ml) return OFB_EINVAL;
    RP_LAUNCH((relpos_fwd_kernel<DT, DP, POS, true>), dim3((unsigned)wgs, splits), lds, s, a);
    const int64_t rows = (int64_t)a.B * a.H * a.Nq;
    hipLaunchKernelGGL((relpos_join_kernel<DT>), dim3((unsigned)((rows + 3) / 4)), dim3(RP_THREADS), 0, s, a, splits);
  } else {
    RP_LAUNCH((relpos_fwd_kernel<DT, DP, POS, false>), dim3((unsigned)wgs), lds, s, a);
  }
  return ofb_launch_status();
}

// 16-bit dQ with heads over 64, where there is at most one workgroup a CU (causal: half as many again, the short ones run behind each other): nothing is
// lost if it takes more than half the registers, so nothing spills and a tile holds 64 keys, not 32.  Step with and without, heads of 128, 8 of them, causal: 2 x 1025
// tokens 174 and 192 us, 4 x 1025 184 and 205, 6 x 1025 230 and 231, 8 x 1025 281 and 259; not causal: 2 x 1025 257 and 273, 4 x 1025 392 and 384.
bool rp_few(const ofb_relpos_args& a) { return (int64_t)a.B * a.H * ((a.Nq + RP_TILE - 1) / RP_TILE) <= (a.causal ? 384 : 256); }

template <int DT, int DP, bool POS> int rp_backward_of(const ofb_relpos_args& a, hipStream_t s) {
  const int nqt = (a.Nq + RP_TILE - 1) / RP_TILE, nkt = (a.Nk + RP_TILE - 1) / RP_TILE;
  const dim3 grid((unsigned)((int64_t)a.B * a.H * nqt));
  if constexpr (DT != RP_F32 && DP > 64) {
    if (rp_few(a)) RP_LAUNCH((relpos_dq_kernel<DT, DP, POS, true>), grid, (rp_lds<DT, DP, 3>(a)), s, a);
    else RP_LAUNCH((relpos_dq_kernel<DT, DP, POS, false>), grid, (rp_lds<DT, DP, 1>(a)), s, a);
  } else {
    RP_LAUNCH((relpos_dq_kernel<DT, DP, POS, false>), grid, (rp_lds<DT, DP, 1>(a)), s, a);
  }
  RP_LAUNCH((relpos_dkv_kernel<DT, DP, POS>), dim3((unsigned)((int64_t)a.B * a.H * nkt)), (rp_lds<DT, DP, 2>(a)), s, a);
  if (a.dtable) {
    hipLaunchKernelGGL(relpos_table_kernel, dim3((unsigned)((int64_t)a.n_buckets * a.H)), dim3(RP_THREADS), 0, s, a, rp_table_rows(a),
                       a.pos_k ? (int64_t)0 : (int64_t)a.B * nqt * 4);
  }
  return ofb_launch_status();
}

template <int DT, int DP> int rp_forward(const ofb_relpos_args& a, hipStream_t s) { return a.pos_k ? rp_forward_of<DT, DP, true>(a, s) : rp_forward_of<DT, DP, false>(a, s); }
template <int DT, int DP> int rp_backward(const ofb_relpos_args& a, hipStream_t s) { return a.pos_k ? rp_backward_of<DT, DP, true>(a, s) : rp_backward_of<DT, DP, false>(a, s); }

#define RP_BY_TYPE(fn, a, s)                                                                                          \
  switch ((a).dtype * 3 + ((a).d <= 32 ? 0 : (a).d <= 64 ? 1 : 2)) {                                                  \
    case 0: return fn<RP_F32, 32>(a, s);                                                                              \
    case 1: return fn<RP_F32, 64>(a, s);                                                                              \
    case 2: return fn<RP_F32, 128>(a, s);                                                                             \
    case 3: return fn<RP_BF16, 32>(a, s);                                                                             \
    case 4: return fn<RP_BF16, 64>(a, s);                                                                             \
    case 5: return fn<RP_BF16, 128>(a, s);                                                                            \
    case 6: return fn<RP_F16, 32>(a, s);                                                                              \
    case 7: return fn<RP_F16, 64>(a, s);                                                                              \
    default: return fn<RP_F16, 128>(a, s);                                                                            \
  }

}  // namespace

extern "C" int ofb_relpos_sizes(const ofb_relpos_args* a, int64_t* out6) {
  if (!a || !out6 || a->B < 1 || a->H < 1 || a->Nq < 1 || a->Nk < 1 || a->width < 1) return OFB_EINVAL;
  const int64_t rows = (int64_t)a->B * a->H * a->Nq, splits = rp_splits(*a);
  out6[0] = splits > 1 ? splits * rows * a->d : 0;             // split_o
  out6[1] = splits > 1 ? splits * rows * 2 : 0;                // split_ml
  out6[2] = (int64_t)a->H * a->width * rp_table_rows(*a);      // partial
  out6[3] = a->pos_k ? 0 : (int64_t)a->H * 2 * a->B * ((a->Nq + RP_TILE - 1) / RP_TILE) * 4;        // sat
  out6[4] = (int64_t)a->B * a->H * ((a->Nq + RP_TILE - 1) / RP_TILE);        // bound_q, bound_do
  out6[5] = rp_own_bounds(*a);
  return OFB_OK;
}

extern "C" int ofb_relpos_amax(const ofb_relpos_args* a, int32_t first, int32_t count, void* stream) {
  if (!a || first < 0 || count < 1 || first + count > 2) return OFB_EINVAL;
  if (a->B < 1 || a->H < 1 || a->Nq < 1 || a->Nk < 1 || a->d < 8 || a->d % 8 || (a->dtype != RP_F32 && a->dtype != RP_F16)) return OFB_EINVAL;
  const int64_t t[2][3] = {{a->k_sb, a->k_st, a->k_sh}, {a->v_sb, a->v_st, a->v_sh}}, unit = a->dtype == RP_F32 ? 4 : 8;
  for (int i = first; i < first + count; ++i) {
    const void* x = i ? a->v : a->k;
    if (!x || !(i ? a->bound_v : a->bound_k) || !ofb_aligned16(x)) return OFB_EINVAL;
    for (int64_t s : t[i])
      if (s % unit || s < 0) return OFB_EINVAL;
  }
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid(RP_NBOUND, count);
  if (a->dtype == RP_F32) hipLaunchKernelGGL((relpos_amax_kernel<RP_F32>), grid, dim3(RP_THREADS), 0, s, *a, first);
  else hipLaunchKernelGGL((relpos_amax_kernel<RP_F16>), grid, dim3(RP_THREADS), 0, s, *a, first);
  return ofb_launch_status();
}

extern "C" int ofb_relpos_fwd(const ofb_relpos_args* a, void* stream) {
  if (const int rc = rp_check(a)) return rc;
  if (a->dtype == RP_F32 && (a->n_bound ? !a->bound_k || !a->bound_v : !rp_own_bounds(*a) || !a->bound_k != !a->bound_v)) return OFB_EINVAL;
  if (!a->out || !ofb_aligned16(a->out) || (a->out32 && !ofb_aligned16(a->out32))) return OFB_EINVAL;
  for (int64_t s : {a->o_sb, a->o_st, a->o_sh})
    if (s % 4 || s < 0) return OFB_EINVAL;
  RP_BY_TYPE(rp_forward, *a, (hipStream_t)stream)
}

extern "C" int ofb_relpos_bwd(const ofb_relpos_args* a, void* stream) {
  if (const int rc = rp_check(a)) return rc;
  if (!a->dout || !a->out32 || !a->stats || !a->delta || !a->dq || !a->dk || !a->dv) return OFB_EINVAL;
  if (a->dtable && (int64_t)a->n_buckets * a->H >= (1 << 24)) return OFB_ELIMIT;
  if (a->dtable && (!a->partial || !a->bucket_start || !a->bucket_order || (!a->pos_k && !a->sat))) return OFB_EINVAL;
  if (a->dtype != RP_BF16 && (!a->bound_v || !a->bound_do || a->n_bound < 1)) return OFB_EINVAL;
  if (a->dtype == RP_F32 && (!a->bound_q || !a->bound_k)) return OFB_EINVAL;
  for (const void* p : {(const void*)a->dout, (const void*)a->out32, (const void*)a->dq, (const void*)a->dk, (const void*)a->dv})
    if (!ofb_aligned16(p)) return OFB_EINVAL;
  const int64_t unit = a->dtype == RP_F32 ? 4 : 8;
  for (int64_t s : {a->do_sb, a->do_st, a->do_sh})
    if (s % unit || s < 0) return OFB_EINVAL;
  for (int64_t s : {a->dq_sb, a->dq_st, a->dq_sh, a->dk_sb, a->dk_st, a->dk_sh, a->dv_sb, a->dv_st, a->dv_sh})
    if (s % 4 || s < 0) return OFB_EINVAL;
  RP_BY_TYPE(rp_backward, *a, (hipStream_t)stream)
}
