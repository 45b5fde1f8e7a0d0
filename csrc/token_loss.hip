// apex_amd._token_loss — losses on the log-probabilities of given tokens.
//
// For a row x of logits (V values), its label y and a temperature T
//   lp = x_y / T - log sum_v exp(x_v / T)
// and for any loss of the lp with c = dloss/dlp
//   dloss/dx_v = c ([v = y] - exp(x_v / T - lse)) / T.
// So every loss here is a pass over the rows that keeps two floats of each
// (its maximum m and log2 of sum exp((x - m) / T)), a small pass over the rows'
// lp that makes the loss and c, and a backward pass that reads the logits again
// and writes their gradient. Rows whose label is `ignore` are not read; their lp
// is 0 and their gradient rows are 0. A label outside [0, V) reads nothing and
// gives NaN. Rows whose gradient is 0 (a clipped token, a weight of 0) are not
// read in the backward pass either.
//
// What bounds them: HBM. Forward reads the labelled rows once (32768 x 50304 bf16,
// 18938 labelled: 281 us, 6.8 TB/s), backward reads them once more and writes the
// whole gradient (880 us, 5.9 TB/s; a large copy by the library moves 5.0). The
// second read is the price of a coefficient that hangs on all rows; where it does
// not, policy_loss can hold a row in registers between its two uses.
#include "common.h"

#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <cmath>
#include <limits>
#include <tuple>
#include <vector>

// All in one file: nothing is called from elsewhere but through the module.
namespace {

// Rows of a tensor [.., V] whose leading dimensions come down to two.
struct Rows {
  long inner, outer_stride, inner_stride;  // row r is at (r / inner) * outer_stride + (r % inner) * inner_stride
  __device__ __forceinline__ long at(long r) const {
    return (r / inner) * outer_stride + (r % inner) * inner_stride;
  }
};

// Sequences over the rows: `length` rows each, or rows [cu[s], cu[s + 1]) where cu is given.
struct Sequences {
  const int* cu;
  long length, rows;
  __device__ __forceinline__ void span(long s, long& begin, long& end) const {
    if (cu) {  // the values cannot be looked at on the host without waiting: keep them inside the rows here
      begin = min(max((long)cu[s], 0L), rows);
      end = min(max((long)cu[s + 1], begin), rows);
    } else {
      begin = s * length;
      end = begin + length;
    }
  }
};

// The sequence of a row, -1 where none has it (cu does not fall)
__device__ __forceinline__ long owner_of(const Sequences& seqs, long count, long row) {
  if (!seqs.cu) return row / seqs.length;
  long lo = 0, hi = count - 1;  // the last one that begins at or before the row
  while (lo < hi) {
    const long mid = (lo + hi + 1) >> 1;
    if (seqs.cu[mid] <= row) lo = mid; else hi = mid - 1;
  }
  long begin, end;
  seqs.span(lo, begin, end);
  return row >= begin && row < end ? lo : -1;
}

template <typename T>
struct Pack {
  static constexpr int width = 16 / sizeof(T);
  T a[width];
};

// A row in packs that are aligned at `p`, and the elements before and behind them:
// rows of an odd V begin anywhere, and packs that lie across cache lines cost
// (rows of 50257 bf16, loads and stores: 5.4 TB/s, of 50304 6.1).
struct Packs {
  int head, whole, singles;  // elements before, packs, elements before and behind
  template <typename T>
  __device__ __forceinline__ static Packs of(const T* p, long V) {
    constexpr int W = 16 / sizeof(T);
    const int head = (int)min((long)((16 - ((unsigned long)p & 15)) & 15) / (long)sizeof(T), V);
    const int whole = (int)((V - head) / W);
    return {head, whole, (int)(V - (long)whole * W)};
  }
  // the element of single j, and whether (and where) the label is one
  __device__ __forceinline__ int single(int j, int W) const { return j < head ? j : whole * W + j; }
  __device__ __forceinline__ bool is_single(long y, int W) const { return y < head || y >= head + (long)whole * W; }
};

// 16 bytes at an address that is aligned to its element only (rows that lie
// otherwise than the gradient's), past the caches: nothing here is met twice in a
// pass
typedef unsigned wide __attribute__((ext_vector_type(4)));
typedef unsigned wide_at_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned wide_at_2 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T>
__device__ __forceinline__ wide load_wide(const T* p) {
  if constexpr (sizeof(T) == 4) return __builtin_nontemporal_load((const wide_at_4*)p);
  else return __builtin_nontemporal_load((const wide_at_2*)p);
}

template <typename T>
__device__ __forceinline__ Pack<T> pack_of(wide v) {
  Pack<T> r;
  __builtin_memcpy(&r, &v, 16);
  return r;
}

template <typename T>
__device__ __forceinline__ Pack<T> load16(const T* p) {
  return pack_of<T>(load_wide(p));
}

template <typename T>
__device__ __forceinline__ void store16(T* p, const Pack<T>& r) {
  wide v;
  __builtin_memcpy(&v, &r, 16);
  if constexpr (sizeof(T) == 4) __builtin_nontemporal_store(v, (wide_at_4*)p);
  else __builtin_nontemporal_store(v, (wide_at_2*)p);
}

// A pack of rounded floats. bf16 goes by the hardware's conversion of pairs: the
// library's, in integer steps, takes as many instructions as all the rest.
template <typename T>
__device__ __forceinline__ Pack<T> rounded(const float* f) {
  Pack<T> r;
#pragma unroll
  for (int j = 0; j < Pack<T>::width; ++j) r.a[j] = from_float<T>(f[j]);
  return r;
}
template <>
__device__ __forceinline__ Pack<__hip_bfloat16> rounded<__hip_bfloat16>(const float* f) {
  typedef float float8 __attribute__((ext_vector_type(8)));
  typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
  float8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = f[j];
  const bf16x8 b = __builtin_convertvector(v, bf16x8);
  Pack<__hip_bfloat16> r;
  __builtin_memcpy(&r, &b, 16);
  return r;
}

// log2(e) / T in two parts: in one, every term of a row's sum is off to the same
// side, and so is the sum of an answer's hundreds of log-probabilities. Both parts
// are over 0, so that a difference of -inf stays one.
struct Base {
  float hi, lo;
  __device__ __forceinline__ float exp(float d) const { return __builtin_amdgcn_exp2f(fmaf(d, hi, d * lo)); }
};

// op over each N neighbouring lanes, on all of them, without LDS: exchanges within
// quads, mirrored halves and rows of 16, then between rows and halves of the wave.
// Lanes of a group hold the same value before they meet another group, so that a
// mirror is an exchange.
template <int CTRL>
__device__ __forceinline__ float lane_across(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ double lane_across(double v) {
  return __hiloint2double(__builtin_amdgcn_mov_dpp(__double2hiint(v), CTRL, 0xF, 0xF, true),
                          __builtin_amdgcn_mov_dpp(__double2loint(v), CTRL, 0xF, 0xF, true));
}
template <bool HALVES>
__device__ __forceinline__ void swap_rows(unsigned v, unsigned& a, unsigned& b) {
  const auto r = HALVES ? __builtin_amdgcn_permlane32_swap(v, v, false, false) : __builtin_amdgcn_permlane16_swap(v, v, false, false);
  a = r[0];
  b = r[1];
}
template <bool HALVES, typename F>
__device__ __forceinline__ float over_rows(float v, F op) {
  unsigned a, b;
  swap_rows<HALVES>(__float_as_uint(v), a, b);
  return op(__uint_as_float(a), __uint_as_float(b));
}
template <bool HALVES, typename F>
__device__ __forceinline__ double over_rows(double v, F op) {
  unsigned ah, bh, al, bl;
  swap_rows<HALVES>(__double2hiint(v), ah, bh);
  swap_rows<HALVES>(__double2loint(v), al, bl);
  return op(__hiloint2double(ah, al), __hiloint2double(bh, bl));
}
template <int N, typename V, typename F>
__device__ __forceinline__ V over_lanes(V v, F op) {
  if constexpr (N >= 2) v = op(v, lane_across<0xB1>(v));    // quad_perm 1,0,3,2
  if constexpr (N >= 4) v = op(v, lane_across<0x4E>(v));    // quad_perm 2,3,0,1
  if constexpr (N >= 8) v = op(v, lane_across<0x141>(v));   // row_half_mirror
  if constexpr (N >= 16) v = op(v, lane_across<0x140>(v));  // row_mirror
  if constexpr (N >= 32) v = over_rows<false>(v, op);
  if constexpr (N >= 64) v = over_rows<true>(v, op);
  return v;
}

// m = max x, s = sum exp((x - m) / T), over what has been added. A pack's few terms
// are added in 32 bits, packs and lanes in 64: half a step off in each of some
// twenty sums of every row shows in the small difference of two answers' hundreds
// of log-probabilities.
struct Running {
  float m = -INFINITY;
  double s = 0;
  // differences are taken from 0 where all so far is -inf: exp of -inf is 0
  __device__ __forceinline__ float origin() const { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void raise(float top, Base c) {
    if (top > m) {
      s *= c.exp(m - top);
      m = top;
    }
  }
  __device__ __forceinline__ void join(float mb, double sb, Base c) {
    const float ma = m;
    m = fmaxf(m, mb);
    const float o = origin();
    s = s * c.exp(ma - o) + sb * c.exp(mb - o);
  }
  // over each N neighbouring lanes, on all of them
  template <int N>
  __device__ __forceinline__ void join_lanes(Base c) {
    const float ma = m;
    m = over_lanes<N>(m, [](float a, float b) { return fmaxf(a, b); });
    s = over_lanes<N>(s * c.exp(ma - origin()), [](double a, double b) { return a + b; });
  }
};

template <int BLOCK>
__device__ __forceinline__ Running block_join(Running w, Base c, double* smem) {
  constexpr int NW = BLOCK / WAVE_SIZE;
  w.join_lanes<WAVE_SIZE>(c);
  if (NW == 1) return w;
  if ((threadIdx.x & (WAVE_SIZE - 1)) == 0) {
    smem[2 * (threadIdx.x / WAVE_SIZE)] = w.m;
    smem[2 * (threadIdx.x / WAVE_SIZE) + 1] = w.s;
  }
  __syncthreads();
  w.m = (float)smem[2 * (threadIdx.x & (NW - 1))];
  w.s = smem[2 * (threadIdx.x & (NW - 1)) + 1];
  w.join_lanes<NW>(c);
  return w;
}

// U packs into the running maximum and sum: one rescaling for all of them
template <typename T, int U>
__device__ __forceinline__ void take(Running& w, const Pack<T>* v, Base c) {
  constexpr int W = Pack<T>::width;
  float top = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < W; ++j) top = fmaxf(top, to_float(v[u].a[j]));
  w.raise(top, c);
  const float o = w.origin();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float part[W];
#pragma unroll
    for (int j = 0; j < W; ++j) part[j] = c.exp(to_float(v[u].a[j]) - o);
    // by halves: a term meets two or three sums
#pragma unroll
    for (int half = W / 2; half > 0; half /= 2)
#pragma unroll
      for (int j = 0; j < half; ++j) part[j] += part[j + half];
    w.s += part[0];
  }
}

__device__ __forceinline__ float log_prob(float x, Running w, double inv_t, float log2s) {
  return (float)((double)(x - w.m) * inv_t - 0.6931471805599453 * (double)log2s);
}

// What a row's pass leaves: its statistics, and its log-probability in 32 bits, or
// in 64 where many of them are going to be added and a small difference of the
// sums is asked for.
struct RowOut {
  float2* stats;
  float* lp;
  double* lp64;
  __device__ __forceinline__ void none(long row, float value) const {
    stats[row] = make_float2(value, value);
    if (lp64) lp64[row] = value;
    else lp[row] = value;
  }
  __device__ __forceinline__ void put(long row, float x, Running w, double inv_t) const {
    const float l2 = log2f((float)w.s);
    stats[row] = make_float2(w.m, l2);
    if (lp64) lp64[row] = (double)(x - w.m) * inv_t - log(w.s);
    else lp[row] = log_prob(x, w, inv_t, l2);
  }
};

// A block's sums of N values in 64 bits, in a fixed order; valid on every thread.
template <int BLOCK, int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double* smem /* N * waves */) {
  constexpr int NW = BLOCK / WAVE_SIZE;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int off = WAVE_SIZE / 2; off > 0; off >>= 1) v[n] += __shfl_xor(v[n], off);
  __syncthreads();  // of what was read from smem before
  if ((threadIdx.x & (WAVE_SIZE - 1)) == 0)
#pragma unroll
    for (int n = 0; n < N; ++n) smem[n * NW + threadIdx.x / WAVE_SIZE] = v[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) v[n] += smem[n * NW + i];
  }
}

// ---------------- rows: maximum, sum and log-probability ----------------
constexpr int UNROLL = 4;  // packs of a lane that are on their way together

template <typename T, int BLOCK>
__global__ void __launch_bounds__(BLOCK) row_stats_kernel(
    const T* __restrict__ logits, Rows where, const long* __restrict__ labels, long ignore, long V,
    long rows, Base c, double inv_t, RowOut out, int* __restrict__ arrived) {
  __shared__ double smem[2 * (BLOCK / WAVE_SIZE)];
  constexpr int W = Pack<T>::width;
  if (arrived && blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;  // for the kernel after this one
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const long y = labels[row];
    if (y == ignore || y < 0 || y >= V) {
      if (threadIdx.x == 0) out.none(row, y == ignore ? 0.f : NAN);
      continue;
    }
    const T* first = logits + where.at(row);
    const Packs in = Packs::of(first, V);
    const T* x = first + in.head;
    const int whole = in.whole;
    Running w;
    T single = from_float<T>(-INFINITY);
    if ((int)threadIdx.x < in.singles) single = first[in.single(threadIdx.x, W)];
    int k = threadIdx.x;
    for (; k + (UNROLL - 1) * BLOCK < whole; k += UNROLL * BLOCK) {
      Pack<T> v[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) v[u] = load16(x + (k + u * BLOCK) * W);
      take<T, UNROLL>(w, v, c);
    }
    if (k < whole) {
      Pack<T> v[UNROLL - 1];
#pragma unroll
      for (int u = 0; u < UNROLL - 1; ++u) v[u] = load16(x + min(k + u * BLOCK, whole - 1) * W);
#pragma unroll
      for (int u = 0; u < UNROLL - 1; ++u)
        if (k + u * BLOCK < whole) take<T, 1>(w, v + u, c);
    }
    w.raise(to_float(single), c);
    w.s += c.exp(to_float(single) - w.origin());
    w = block_join<BLOCK>(w, c, smem);
    if (threadIdx.x == 0) out.put(row, to_float(first[y]), w, inv_t);
    __syncthreads();  // smem is the next row's
  }
}

// Few long rows: a block has UNROLL packs of each lane, a second kernel joins a
// row's parts. Along grid.x are the parts of a row.
constexpr int PART_BLOCK = 256, PART_PACKS = PART_BLOCK * UNROLL;

template <typename T>
__global__ void __launch_bounds__(PART_BLOCK) row_part_kernel(
    const T* __restrict__ logits, Rows where, const long* __restrict__ labels, long ignore, long V, Base c,
    float2* __restrict__ parts, int* __restrict__ arrived) {
  __shared__ double smem[2 * (PART_BLOCK / WAVE_SIZE)];
  constexpr int W = Pack<T>::width;
  const long row = blockIdx.y, whole = V / W;
  if (arrived && blockIdx.x + blockIdx.y == 0 && threadIdx.x == 0) *arrived = 0;  // for the kernel after the next
  if (labels[row] == ignore) return;
  const T* x = logits + where.at(row);
  Running w;
  const long k = (long)blockIdx.x * PART_PACKS + threadIdx.x;
  Pack<T> v[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u)
    if (k + u * PART_BLOCK < whole) v[u] = load16(x + (k + u * PART_BLOCK) * W);
#pragma unroll
  for (int u = 0; u < UNROLL; ++u)
    if (k + u * PART_BLOCK < whole) take<T, 1>(w, v + u, c);
  if (const long i = whole * W + threadIdx.x; blockIdx.x == gridDim.x - 1 && i < V) {
    const float f = to_float(x[i]);
    w.raise(f, c);
    w.s += c.exp(f - w.origin());
  }
  w = block_join<PART_BLOCK>(w, c, smem);
  if (threadIdx.x == 0) parts[row * gridDim.x + blockIdx.x] = make_float2(w.m, (float)w.s);
}

template <typename T>
__global__ void __launch_bounds__(WAVE_SIZE) row_join_kernel(
    const T* __restrict__ logits, Rows where, const long* __restrict__ labels, long ignore, long V, Base c,
    double inv_t, const float2* __restrict__ parts, int count, RowOut out) {
  const long row = blockIdx.x, y = labels[row];
  if (y == ignore || y < 0 || y >= V) {
    if (threadIdx.x == 0) out.none(row, y == ignore ? 0.f : NAN);
    return;
  }
  const float xy = to_float(logits[where.at(row) + y]);
  Running w;
  for (int i = threadIdx.x; i < count; i += WAVE_SIZE) {
    const float2 part = parts[row * count + i];
    w.join(part.x, part.y, c);
  }
  w.join_lanes<WAVE_SIZE>(c);
  if (threadIdx.x == 0) out.put(row, xy, w, inv_t);
}

// ---------------- rows: gradient ----------------
template <typename T>
__device__ __forceinline__ Pack<T> zeros() {
  Pack<T> z;
#pragma unroll
  for (int j = 0; j < Pack<T>::width; ++j) z.a[j] = from_float<T>(0.f);
  return z;
}

// A row's f ([v = y] - p), p = exp2((x - m) c - log2 s)
struct Gradient {
  float f, m, l2, c;
  __device__ __forceinline__ float p(float x) const { return __builtin_amdgcn_exp2f(fmaf(x - m, c, -l2)); }
  __device__ __forceinline__ float at_label(float x) const { return f * (1.f - p(x)); }
  // a pack as if it had no label
  template <typename T>
  __device__ __forceinline__ void put(const Pack<T>& v, T* g) const {
    constexpr int W = Pack<T>::width;
    float o[W];
#pragma unroll
    for (int j = 0; j < W; ++j) o[j] = -f * p(to_float(v.a[j]));
    store16(g, rounded<T>(o));
  }
};

// coef[r] (with `scale` and `norm`, where given) is the gradient of row r's lp.
// A block has one pack of each lane: grid.x goes along the row, grid.y over rows.
// Blocks that take more of a row, or all of it, are slower: the bare accesses of
// 32768 x 50304 bf16 take 831 us so, 953 by four packs a lane, 995 by a row a
// block; with loads and stores through the caches 904, 983 and 1005.
// 256 threads: the whole policy loss of that size takes 1175 us, with 64 1249,
// 128 1180, 512 1268, 1024 1412; with half as many blocks on a compute unit 1536.
template <typename T, int BLOCK>
__global__ void __launch_bounds__(BLOCK) row_grad_kernel(
    const T* __restrict__ logits, Rows where, const long* __restrict__ labels, long ignore, long V,
    long rows, float c, float inv_t, const float2* __restrict__ stats, const float* __restrict__ coef,
    const float* __restrict__ scale, long scale_stride, const float* __restrict__ norm,
    T* __restrict__ grad) {
  constexpr int W = Pack<T>::width;
  const int k = blockIdx.x * BLOCK + threadIdx.x;
  for (long row = blockIdx.y; row < rows; row += gridDim.y) {
    const long y = labels[row];
    T* g = grad + row * V;
    const Packs in = Packs::of(g, V);
    // the row's first lanes have the elements that make no pack as well
    const bool pack = k < in.whole, one = k < in.singles;
    const int i = in.head + k * W, single = in.single(k, W);
    float f = coef[row] * inv_t;
    if (scale) f *= scale[row * scale_stride];
    if (norm) f *= *norm;
    if (y == ignore || f == 0.f) {  // a clipped token, or one that no sequence has: its logits are not asked
      if (pack) store16(g + i, zeros<T>());
      if (one) g[single] = from_float<T>(0.f);
      continue;
    }
    const T* x = logits + where.at(row);
    const float2 st = stats[row];
    const Gradient d{f, st.x, st.y, c};
    if (pack) d.put(load16(x + i), g + i);
    if (one) g[single] = from_float<T>(-f * d.p(to_float(x[single])));
    // the label's element, by the lane that has just written its pack
    if (y >= 0 && y < V && ((pack && y >= i && y < i + W) || (one && y == single)))
      g[y] = from_float<T>(d.at_label(to_float(x[y])));
  }
}

// ---------------- sequences ----------------
// A block has a sequence (or a pair): 256 threads, or 1024 where sequences are long.

// A lane's sum (in 64 bits) and number of a sequence's labelled lp.
template <int BLOCK>
__device__ __forceinline__ void sum_span(const double* lp, const long* labels, long ignore, long begin,
                                         long end, double& sum, double& count) {
  sum = count = 0;
#pragma unroll 2
  for (long r = begin + threadIdx.x; r < end; r += BLOCK) {
    const double v = lp[r];
    const bool on = labels[r] != ignore;
    sum += on ? v : 0.0;
    count += on ? 1.0 : 0.0;
  }
}

template <int BLOCK>
__global__ void __launch_bounds__(BLOCK) sequence_sum_kernel(
    const double* __restrict__ lp, const long* __restrict__ labels, long ignore, Sequences seqs,
    bool average, float* __restrict__ out) {
  __shared__ double smem[2 * BLOCK / WAVE_SIZE];
  long begin, end;
  seqs.span(blockIdx.x, begin, end);
  double v[2];  // sum and number
  sum_span<BLOCK>(lp, labels, ignore, begin, end, v[0], v[1]);
  block_sums<BLOCK>(v, smem);
  if (threadIdx.x == 0) out[blockIdx.x] = (float)(average ? v[0] / fmax(v[1], 1.0) : v[0]);
}

// coef of each row of a sequence from the gradient of the sequence's sum
template <int BLOCK>
__global__ void __launch_bounds__(BLOCK) sequence_coef_kernel(
    const float* __restrict__ grad, const long* __restrict__ labels, long ignore, Sequences seqs,
    bool average, float* __restrict__ coef) {
  __shared__ double smem[BLOCK / WAVE_SIZE];
  long begin, end;
  seqs.span(blockIdx.x, begin, end);
  double n[1] = {0};
  if (average) {
    for (long r = begin + threadIdx.x; r < end; r += BLOCK) n[0] += labels[r] != ignore ? 1.0 : 0.0;
    block_sums<BLOCK>(n, smem);
  }
  const float f = average ? (float)(grad[blockIdx.x] / fmax(n[0], 1.0)) : grad[blockIdx.x];
  for (long r = begin + threadIdx.x; r < end; r += BLOCK) coef[r] = f;
}

// True on the block that comes last, on all its threads; what the others wrote before is then visible to it.
__device__ __forceinline__ bool comes_last(int* arrived, int blocks, int* smem) {
  if (threadIdx.x == 0) {
    __threadfence();
    *smem = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == blocks - 1;
    __threadfence();
  }
  __syncthreads();
  return *smem != 0;
}

__device__ __forceinline__ double read_shared(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------- paired log ratios ----------------
// One block a pair: sequence b was chosen, sequence pairs + b rejected. With
// d = (S_chosen - R_chosen) - (S_rejected - R_rejected), S and R the sequences'
// log-probabilities under the policy and the reference:
//   sigmoid: -(1 - e) log sigmoid(beta d) - e log sigmoid(-beta d)
//   ipo:     (d - 1 / (2 beta))^2
//   hinge:   max(0, 1 - beta d)
// The sums and d are kept in 64 bits: d is a small difference of large sums.
enum { SIGMOID = 0, IPO = 1, HINGE = 2 };

template <int BLOCK>
__global__ void __launch_bounds__(BLOCK) preference_kernel(
    const double* __restrict__ lp, const long* __restrict__ labels, long ignore, Sequences seqs,
    const float* __restrict__ ref, long pairs, int kind, double beta, double smoothing, bool average,
    float* __restrict__ coef, float* __restrict__ chosen_out, float* __restrict__ rejected_out,
    double* __restrict__ partial, int* __restrict__ arrived, float* __restrict__ loss_out) {
  __shared__ double smem[4 * BLOCK / WAVE_SIZE];
  __shared__ int last;
  const long b = blockIdx.x;
  long begin[2], end[2];
  double v[4], count[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    seqs.span(b + k * pairs, begin[k], end[k]);
    sum_span<BLOCK>(lp, labels, ignore, begin[k], end[k], v[k], v[2 + k]);
  }
  const double ref_chosen = ref[b], ref_rejected = ref[b + pairs];
  block_sums<BLOCK>(v, smem);
#pragma unroll
  for (int k = 0; k < 2; ++k) count[k] = average ? fmax(v[2 + k], 1.0) : 1.0;
  const double chosen = v[0] / count[0] - ref_chosen;
  const double rejected = v[1] / count[1] - ref_rejected;
  const double d = chosen - rejected, z = beta * d;
  double loss, slope;  // slope = dloss/dd
  if (kind == SIGMOID) {
    // log(1 + exp(-z)) without an exp that overflows
    const double e = exp(-fabs(z)), soft = log1p(e);
    const double minus = fmax(-z, 0.0) + soft, plus = fmax(z, 0.0) + soft;
    const double up = (z >= 0 ? e : 1.0) / (1.0 + e);  // sigmoid(-z)
    loss = (1.0 - smoothing) * minus + (smoothing > 0 ? smoothing * plus : 0.0);  // plus may be infinite
    slope = beta * (smoothing * (1.0 - up) - (1.0 - smoothing) * up);
  } else if (kind == IPO) {
    const double off = d - 0.5 / beta;
    loss = off * off;
    slope = 2.0 * off;
  } else {
    loss = z >= 1.0 ? 0.0 : 1.0 - z;  // NaN stays NaN
    slope = z >= 1.0 ? 0.0 : -beta;
  }
  slope = z != z ? z : slope;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float f = (float)((k ? -slope : slope) / (count[k] * (double)pairs));
    for (long r = begin[k] + threadIdx.x; r < end[k]; r += BLOCK) coef[r] = f;
  }
  if (threadIdx.x == 0) {
    chosen_out[b] = (float)(beta * chosen);
    rejected_out[b] = (float)(beta * rejected);
    partial[b] = loss;
  }
  if (!comes_last(arrived, gridDim.x, &last)) return;
  double total[1] = {0};
  for (long i = threadIdx.x; i < pairs; i += BLOCK) total[0] += read_shared(partial + i);
  block_sums<BLOCK>(total, smem);
  if (threadIdx.x == 0) *loss_out = (float)(total[0] / (double)pairs);
}

// ---------------- clipped policy loss ----------------
// With ratio = exp(lp - old), advantage A and d = ref - lp:
//   loss = -min(ratio A, clamp(ratio, 1 - low, 1 + high) A) + kl (exp(d) - d - 1)
//   dloss/dlp = (-ratio A where the minimum is the unclipped one) - kl (exp(d) - 1)
struct Policy {
  const float *old, *ref, *advantages;
  bool by_row;  // an advantage for each row, or for each sequence
  float low, high, kl;
  __device__ __forceinline__ float of(float lp, long r, long s, float& slope) const {
    const float a = advantages[by_row ? r : s];
    const float ratio = old ? expf(lp - old[r]) : (lp == lp ? 1.f : lp);
    const float held = ratio < 1.f - low ? 1.f - low : ratio > 1.f + high ? 1.f + high : ratio;
    float loss = -(ratio * a > held * a ? held * a : ratio * a);
    slope = ratio * a > held * a ? 0.f : -ratio * a;
    if (ref) {
      const float d = ref[r] - lp, grown = expm1f(d);
      loss = fmaf(kl, grown - d, loss);
      slope = fmaf(-kl, grown, slope);
    }
    return loss;
  }
};

enum { TOKEN = 0, SEQUENCE = 1, SUM = 2, NONE = 3 };

// One block a sequence. `coef` comes without the division by the number of all
// tokens (TOKEN): that number is known at the end only and goes out as `norm`.
template <int BLOCK>
__global__ void __launch_bounds__(BLOCK) policy_kernel(
    const float* __restrict__ lp, const long* __restrict__ labels, long ignore, Sequences seqs,
    Policy policy, int reduction, float* __restrict__ coef, float* __restrict__ losses,
    double* __restrict__ partial, int* __restrict__ arrived, float* __restrict__ norm,
    float* __restrict__ loss_out) {
  __shared__ double smem[2 * BLOCK / WAVE_SIZE];
  __shared__ int last;
  const long s = blockIdx.x;
  long begin, end;
  seqs.span(s, begin, end);
  double weight = 1.0;
  if (reduction == SEQUENCE) {  // its number of tokens has to be known first
    double n[1] = {0};
    for (long r = begin + threadIdx.x; r < end; r += BLOCK) n[0] += labels[r] != ignore ? 1.0 : 0.0;
    block_sums<BLOCK>(n, smem);
    weight = 1.0 / (fmax(n[0], 1.0) * (double)gridDim.x);
  }
  double v[2] = {0, 0};  // loss and number of tokens
  for (long r = begin + threadIdx.x; r < end; r += BLOCK) {
    float loss = 0.f, slope = 0.f;
    if (labels[r] != ignore) {
      loss = policy.of(lp[r], r, s, slope);
      v[1] += 1.0;
    }
    coef[r] = (float)(weight * slope);
    if (reduction == NONE) losses[r] = loss;
    v[0] += weight * loss;
  }
  if (reduction == NONE) return;
  block_sums<BLOCK>(v, smem);
  if (threadIdx.x == 0) {
    partial[2 * s] = v[0];
    partial[2 * s + 1] = v[1];
  }
  if (!comes_last(arrived, gridDim.x, &last)) return;
  v[0] = v[1] = 0;
  for (long i = threadIdx.x; i < gridDim.x; i += BLOCK) {
    v[0] += read_shared(partial + 2 * i);
    v[1] += read_shared(partial + 2 * i + 1);
  }
  block_sums<BLOCK>(v, smem);
  if (threadIdx.x == 0) {
    const double by = reduction == TOKEN ? 1.0 / fmax(v[1], 1.0) : 1.0;
    *norm = (float)by;
    *loss_out = (float)(v[0] * by);
  }
}

// ---------------- policy loss and gradient at once ----------------
// Where the gradient of the loss is known beforehand, a row's logits are read
// once: a block holds them in registers from the first use to the second. 4096 x
// 131072 bf16 (2550 labelled): 336 us, 5.2 TB/s, one row a compute unit; 11920 x
// 50304, all labelled: 431 us, 5.6 TB/s, against 591 in two passes. Blocks that
// stay and load the next row into each pack's registers as soon as that is
// written are slower (16000 wide 437 us for 369): their 16 packs, two rows'
// addresses and the floats in between leave no room for a second row's block.

// What has to be known before: the weight of a token in the loss (of each
// sequence, or weights[0] for all), and what the gradient is multiplied by.
constexpr int PREPARE_BLOCK = 1024;
__global__ void __launch_bounds__(PREPARE_BLOCK) policy_prepare_kernel(
    const long* __restrict__ labels, long ignore, Sequences seqs, long count, int reduction, float number,
    const float* __restrict__ value, float* __restrict__ applied, float* __restrict__ weights,
    int* __restrict__ arrived) {
  __shared__ double smem[PREPARE_BLOCK / WAVE_SIZE];
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *applied = value ? number * *value : number;
    *arrived = 0;
  }
  long begin, end, unused;
  seqs.span(reduction == SEQUENCE ? blockIdx.x : 0, begin, end);
  if (reduction != SEQUENCE) seqs.span(count - 1, unused, end);
  int n = 0;
  if (reduction != SUM) {
#pragma unroll 4
    for (long r = begin + threadIdx.x; r < end; r += PREPARE_BLOCK) n += labels[r] != ignore ? 1 : 0;
  }
  double all[1] = {(double)n};
  block_sums<PREPARE_BLOCK>(all, smem);
  if (threadIdx.x == 0)
    weights[blockIdx.x] = (float)(reduction == SUM ? 1.0 : 1.0 / (fmax(all[0], 1.0) * (reduction == SEQUENCE ? (double)count : 1.0)));
}

// One block a row, at most NP packs a lane and NP - 2 of each at least: only the
// last two are asked for.
template <typename T, int BLOCK, int NP>
__global__ void __launch_bounds__(BLOCK, 4) policy_at_once_kernel(
    const T* __restrict__ logits, Rows where, const long* __restrict__ labels, long ignore, long V, long first_row,
    Base c, double inv_t, Sequences seqs, long count, Policy policy, bool weight_by_sequence,
    const float* __restrict__ weights, const float* __restrict__ applied, float* __restrict__ lp_out,
    float* __restrict__ losses, T* __restrict__ grad) {
  __shared__ double smem[2 * (BLOCK / WAVE_SIZE)];
  constexpr int W = Pack<T>::width;
  const long row = first_row + blockIdx.x;
  const long y = labels[row];
  T* g = grad + row * V;
  const Packs in = Packs::of(g, V);
  const int whole = in.whole, lane = in.head + (int)threadIdx.x * W;
  const bool one = (int)threadIdx.x < in.singles;
  const int single = in.single(threadIdx.x, W);
  const auto put_zeros = [&] {
    for (int k = threadIdx.x; k < whole; k += BLOCK) store16(g + in.head + k * W, zeros<T>());
    if (one) g[single] = from_float<T>(0.f);
  };
  if (y == ignore) {
    if (threadIdx.x == 0) lp_out[row] = losses[row] = 0.f;
    put_zeros();
    return;
  }
  const T* x = logits + where.at(row);
  const bool valid = y >= 0 && y < V;
  const T xy = x[valid ? y : 0];
  const bool has[2] = {(NP - 2) * BLOCK + (int)threadIdx.x < whole, (NP - 1) * BLOCK + (int)threadIdx.x < whole};
  wide v[NP];
#pragma unroll
  for (int u = 0; u < NP; ++u)
    if (u < NP - 2 || has[u - (NP - 2)]) v[u] = load_wide(x + u * BLOCK * W + lane);
  T xt = from_float<T>(-INFINITY);
  if (one) xt = x[single];
  Running w;
#pragma unroll
  for (int u = 0; u < NP; ++u)
    if (u < NP - 2 || has[u - (NP - 2)]) {
      const Pack<T> some = pack_of<T>(v[u]);
      take<T, 1>(w, &some, c);
      __builtin_amdgcn_sched_barrier(0);  // one pack's floats at a time: the packs take half of the registers
    }
  w.raise(to_float(xt), c);
  w.s += c.exp(to_float(xt) - w.origin());
  w = block_join<BLOCK>(w, c, smem);
  const float l2 = log2f((float)w.s), lp = log_prob(valid ? to_float(xy) : NAN, w, inv_t, l2);
  float f = 0.f, loss = 0.f;
  const long s = owner_of(seqs, count, row);
  if (s >= 0) {
    float slope;
    const float weight = weights[weight_by_sequence ? s : 0];
    loss = weight * policy.of(lp, row, s, slope);
    f = weight * slope * *applied * (float)inv_t;
  }
  if (threadIdx.x == 0) {
    lp_out[row] = lp;
    losses[row] = loss;
  }
  if (f == 0.f) {
    put_zeros();
    return;
  }
  const Gradient d{f, w.m, l2, c.hi + c.lo};  // the base rounded to nearest, as row_grad_kernel has it
#pragma unroll
  for (int u = 0; u < NP; ++u)
    if (u < NP - 2 || has[u - (NP - 2)]) {
      // converted again: kept from the first use, the floats would take twice the registers
      asm volatile("" : "+v"(v[u]));
      d.put(pack_of<T>(v[u]), g + u * BLOCK * W + lane);
      __builtin_amdgcn_sched_barrier(0);
    }
  if (one) g[single] = from_float<T>(-f * d.p(to_float(xt)));
  // the label's element, by the lane that has just written its pack
  if (valid && (in.is_single(y, W) ? one && y == single : (y - in.head) / W % BLOCK == threadIdx.x))
    g[y] = from_float<T>(d.at_label(to_float(xy)));
}

// The rows' weighted losses, in a fixed order and 64 bits
constexpr int TOTAL_BLOCK = 1024;
__global__ void __launch_bounds__(TOTAL_BLOCK) total_kernel(const float* __restrict__ losses, long rows,
                                                            double* __restrict__ partial, int* __restrict__ arrived,
                                                            float* __restrict__ loss_out) {
  __shared__ double smem[TOTAL_BLOCK / WAVE_SIZE];
  __shared__ int last;
  double sum[1] = {0};
  for (long r = (long)blockIdx.x * TOTAL_BLOCK + threadIdx.x; r < rows; r += (long)gridDim.x * TOTAL_BLOCK) sum[0] += losses[r];
  block_sums<TOTAL_BLOCK>(sum, smem);
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) partial[blockIdx.x] = sum[0];
    if (!comes_last(arrived, gridDim.x, &last)) return;
    sum[0] = threadIdx.x < gridDim.x ? read_shared(partial + threadIdx.x) : 0.0;
    block_sums<TOTAL_BLOCK>(sum, smem);
  }
  if (threadIdx.x == 0) *loss_out = (float)sum[0];
}

// A gradient made for `applied` becomes that for *scale. Most often they are the same and nothing is moved.
template <typename T>
__global__ void __launch_bounds__(256) rescale_kernel(T* __restrict__ grad, long n, const float* __restrict__ scale,
                                                      const float* __restrict__ applied) {
  const float a = *applied, b = *scale;
  if (a == b) return;
  const float f = b / a;
  constexpr int W = Pack<T>::width;
  const long step = (long)gridDim.x * 256, whole = n / W, first = blockIdx.x * 256L + threadIdx.x;
  for (long k = first; k < whole; k += step) {
    Pack<T> v = load16(grad + k * W);
#pragma unroll
    for (int j = 0; j < W; ++j) v.a[j] = from_float<T>(to_float(v.a[j]) * f);
    store16(grad + k * W, v);
  }
  for (long i = whole * W + first; i < n; i += step) grad[i] = from_float<T>(to_float(grad[i]) * f);
}

// ---------------- host ----------------
Rows rows_of(at::Tensor& x) {
  // merges leading dimensions that lie evenly; copies what does not come down to two
  for (int pass = 0; pass < 2; ++pass) {
    std::vector<std::pair<long, long>> dims;  // (size, stride), outermost first
    for (int64_t d = 0; d + 1 < x.dim(); ++d) {
      if (x.size(d) == 1) continue;
      if (!dims.empty() && dims.back().second == x.stride(d) * x.size(d))
        dims.back() = {dims.back().first * x.size(d), x.stride(d)};
      else
        dims.push_back({x.size(d), x.stride(d)});
    }
    if (dims.size() <= 2 && (x.stride(-1) == 1 || x.size(-1) == 1)) {
      if (dims.empty()) return {1, 0, 0};
      if (dims.size() == 1) return {dims[0].first, 0, dims[0].second};
      return {dims[1].first, dims[0].second, dims[1].second};
    }
    x = x.contiguous();
  }
  TORCH_CHECK(false, "token_loss: logits do not come down to rows");
}

Base base_of(double temperature) {
  const double c = 1.4426950408889634 / temperature;
  float hi = (float)c;
  if (hi > c) hi = std::nextafter(hi, 0.f);
  return {hi, std::max((float)(c - hi), 1e-30f)};
}

// a launch's threads are counted in 32 bits: further rows are taken in turns
unsigned grid_of(long rows) { return (unsigned)std::min<long>(rows, 1 << 20); }

void check_rows(const at::Tensor& logits, const at::Tensor& labels) {
  TORCH_CHECK(logits.is_cuda(), "token_loss: logits must be on the GPU");
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) > 0, "token_loss: logits need a last dimension of the vocabulary");
  TORCH_CHECK(labels.scalar_type() == at::kLong, "token_loss: labels must be int64");
  TORCH_CHECK(labels.device() == logits.device(), "token_loss: labels are on another device than the logits");
  TORCH_CHECK(labels.is_contiguous(), "token_loss: labels must be contiguous");
  TORCH_CHECK(labels.numel() * logits.size(-1) == logits.numel(), "token_loss: one label a row");
  TORCH_CHECK(labels.numel() < std::numeric_limits<int>::max() && logits.size(-1) < (1L << 30), "token_loss: too many rows, or too long ones");
}

// fp32 and contiguous, on the logits' device, with n values
const float* floats(const at::Tensor& t, const at::Tensor& logits, int64_t n, const char* name) {
  TORCH_CHECK(t.device() == logits.device(), "token_loss: ", name, " is on another device than the logits");
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous(), "token_loss: ", name, " must be contiguous fp32");
  TORCH_CHECK(t.numel() == n, "token_loss: ", name, " has ", t.numel(), " values, not ", n);
  return t.data_ptr<float>();
}

Sequences sequences_of(const at::Tensor& labels, const c10::optional<at::Tensor>& cu, long count) {
  TORCH_CHECK(count < (1 << 22), "token_loss: too many sequences");
  Sequences s{nullptr, count ? labels.numel() / count : 0, labels.numel()};
  if (cu) {
    TORCH_CHECK(cu->device() == labels.device() && cu->scalar_type() == at::kInt && cu->is_contiguous(),
                "token_loss: cu_seqlens must be contiguous int32 on the logits' device");
    TORCH_CHECK(cu->numel() == count + 1, "token_loss: cu_seqlens has one value more than sequences");
    s.cu = cu->data_ptr<int>();
  } else {
    TORCH_CHECK(count > 0 ? labels.numel() % count == 0 : labels.numel() == 0, "token_loss: rows do not divide into sequences");
  }
  return s;
}

Policy policy_of(const at::Tensor& logits, const c10::optional<at::Tensor>& old, const at::Tensor& advantages,
                 bool by_row, const c10::optional<at::Tensor>& ref, long rows, long count, double low, double high,
                 double kl) {
  return {old ? floats(*old, logits, rows, "old_log_probs") : nullptr,
          ref ? floats(*ref, logits, rows, "ref_log_probs") : nullptr,
          floats(advantages, logits, by_row ? rows : count, "advantages"), by_row, (float)low, (float)high, (float)kl};
}

// What the backward pass of a loss needs, in one allocation: of each row its
// statistics and its coefficient, and the number that all coefficients are
// multiplied by.
struct Kept {
  at::Tensor room;
  float *stats, *coef, *norm;
  static Kept of(const at::Tensor& room, long rows) {
    float* p = room.data_ptr<float>();
    return {room, p, p + 2 * rows, p + 3 * rows};
  }
  // rows behind the last packed sequence belong to none: no loss, no gradient
  static Kept make(const at::TensorOptions& opts, long rows, bool packed) {
    return of(packed ? at::zeros({3 * rows + 1}, opts) : at::empty({3 * rows + 1}, opts), rows);
  }
};

void launch_stats(at::Tensor logits, const at::Tensor& labels, long ignore, double temperature,
                  float* stats, float* lp, double* lp64, int* arrived) {
  const RowOut out{(float2*)stats, lp, lp64};
  const Rows where = rows_of(logits);
  const long V = logits.size(-1), rows = labels.numel();
  const Base c = base_of(temperature);
  const long* y = labels.data_ptr<long>();
  APEX_DISPATCH_FLOAT_HALF_BF(logits.scalar_type(), "token_loss", ([&] {
    const auto* x = (const scalar_t*)logits.data_ptr();
    const long packs = V / Pack<scalar_t>::width;
    // Up to 64 rows of 128 KB and more leave most of the chip without work: one to 64 rows of 131072 bf16 take 10.0 to
    // 12.4 us by blocks of a row each, 5.5 to 9.7 in parts. At half that length, 5.9 to 7.7 and 5.4 to 8.1, the second
    // launch costs what it saves, and at a quarter more than that.
    if (rows <= 64 && packs >= 8192) {
      const int parts = (int)((packs + PART_PACKS - 1) / PART_PACKS);
      auto room = at::empty({rows * parts, 2}, logits.options().dtype(at::kFloat));
      auto* p = (float2*)room.data_ptr<float>();
      hipLaunchKernelGGL((row_part_kernel<scalar_t>), dim3(parts, rows), dim3(PART_BLOCK), 0, current_stream(), x,
                         where, y, ignore, V, c, p, arrived);
      HIP_CHECK(hipGetLastError());
      hipLaunchKernelGGL((row_join_kernel<scalar_t>), dim3(rows), dim3(WAVE_SIZE), 0, current_stream(), x, where, y,
                         ignore, V, c, 1.0 / temperature, p, parts, out);
      return;
    }
    auto launch = [&](auto block) {
      constexpr int BLOCK = decltype(block)::value;
      hipLaunchKernelGGL((row_stats_kernel<scalar_t, BLOCK>), dim3(grid_of(rows)), dim3(BLOCK), 0, current_stream(),
                         x, where, y, ignore, V, rows, c, 1.0 / temperature, out, arrived);
    };
    // A block's cost is that of its start and of its join, which grow with its waves, and of its passes one after
    // another. 8192 rows of 2048 bf16: 10.3 us by 64 lanes, 14.7 by 128; of 8192: 26.6 by 128, 29.2 by 256; of 32000:
    // 87 by 256, 105 by 512; of 131072: 330 by 256, 319 by 512. Up to 512 rows, two for a compute unit, wait for their
    // passes, not for room: 256 rows of 20000 6.4 by 256, 5.4 by 512, 512 rows 7.5 and 7.2, 640 rows 8.6 and 9.2; of 4800
    // 4.2 and 4.0, 4.5 and 4.6, 4.8 and 6.2.
    using std::integral_constant;
    if (packs <= 512) launch(integral_constant<int, 64>{});
    else if (packs <= 1536 && rows >= 1024) launch(integral_constant<int, 128>{});
    else if (rows > 512 && packs < 8192) launch(integral_constant<int, 256>{});
    else launch(integral_constant<int, 512>{});
  }()));
  HIP_CHECK(hipGetLastError());
}

// Calls launch(block size) for blocks that have a sequence of `rows / count` rows each.
template <typename F>
void by_length(long rows, long count, F launch) {
  if (rows / count > 512) launch(std::integral_constant<int, 1024>{});
  else launch(std::integral_constant<int, 256>{});
}

// -> (lp, stats): stats [rows, 2] is what the backward pass needs of each row
std::tuple<at::Tensor, at::Tensor> token_forward(at::Tensor logits, at::Tensor labels, long ignore,
                                                 double temperature) {
  check_rows(logits, labels);
  const at::DeviceGuard guard(logits.device());
  auto opts = logits.options().dtype(at::kFloat);
  auto lp = at::empty(labels.sizes(), opts);
  auto stats = at::empty({labels.numel(), 2}, opts);
  if (labels.numel())
    launch_stats(logits, labels, ignore, temperature, stats.data_ptr<float>(), lp.data_ptr<float>(), nullptr, nullptr);
  return {lp, stats};
}

// The logits' gradient from that of the rows' log-probabilities: coef, times `scale` (one value, or one a row) and `norm`
at::Tensor rows_backward(at::Tensor logits, const at::Tensor& labels, const float* stats, const float* coef,
                         const at::Tensor& scale, const float* norm, long ignore, double temperature) {
  check_rows(logits, labels);
  const at::DeviceGuard guard(logits.device());
  const long rows = labels.numel(), V = logits.size(-1);
  auto grad = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
  if (!rows) return grad;
  const Rows where = rows_of(logits);
  const float* sc = scale.defined() ? floats(scale, logits, scale.numel() == 1 ? 1 : rows, "grad_output") : nullptr;
  const long step = scale.defined() && scale.numel() == rows && rows > 1 ? 1 : 0;
  APEX_DISPATCH_FLOAT_HALF_BF(logits.scalar_type(), "token_loss", ([&] {
    const long lanes = std::max(V / Pack<scalar_t>::width, 1L);
    auto launch = [&](auto block) {
      constexpr int BLOCK = decltype(block)::value;
      const dim3 grid((lanes + BLOCK - 1) / BLOCK, std::min<long>(rows, 65535));
      hipLaunchKernelGGL((row_grad_kernel<scalar_t, BLOCK>), grid, dim3(BLOCK), 0, current_stream(),
                         (const scalar_t*)logits.data_ptr(), where, labels.data_ptr<long>(), ignore, V, rows,
                         (float)(1.4426950408889634 / temperature), (float)(1.0 / temperature),
                         (const float2*)stats, coef, sc, step, norm, (scalar_t*)grad.data_ptr());
    };
    if (lanes <= 64) launch(std::integral_constant<int, 64>{});
    else if (lanes <= 128) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, 256>{});
  }()));
  HIP_CHECK(hipGetLastError());
  return grad;
}

// -> (sums, stats)
std::tuple<at::Tensor, at::Tensor> sequence_forward(at::Tensor logits, at::Tensor labels,
                                                    c10::optional<at::Tensor> cu, long count, bool average,
                                                    long ignore, double temperature) {
  check_rows(logits, labels);
  const at::DeviceGuard guard(logits.device());
  auto opts = logits.options().dtype(at::kFloat);
  const Sequences seqs = sequences_of(labels, cu, count);
  auto lp = at::empty({labels.numel()}, opts.dtype(at::kDouble));
  auto stats = at::empty({labels.numel(), 2}, opts);
  auto out = at::empty({count}, opts);
  if (labels.numel())
    launch_stats(logits, labels, ignore, temperature, stats.data_ptr<float>(), nullptr, lp.data_ptr<double>(), nullptr);
  if (count)
    by_length(labels.numel(), count, [&](auto block) {
      constexpr int BLOCK = decltype(block)::value;
      hipLaunchKernelGGL((sequence_sum_kernel<BLOCK>), dim3(count), dim3(BLOCK), 0, current_stream(),
                         lp.data_ptr<double>(), labels.data_ptr<long>(), ignore, seqs, average, out.data_ptr<float>());
    });
  HIP_CHECK(hipGetLastError());
  return {out, stats};
}

at::Tensor sequence_coef(at::Tensor grad, at::Tensor labels, c10::optional<at::Tensor> cu, bool average, long ignore) {
  const at::DeviceGuard guard(labels.device());
  const long count = grad.numel();
  const Sequences seqs = sequences_of(labels, cu, count);
  const float* g = floats(grad, labels, count, "grad_output");
  // rows behind the last packed sequence belong to none and get 0
  auto coef = cu ? at::zeros(labels.sizes(), grad.options()) : at::empty(labels.sizes(), grad.options());
  if (count)
    by_length(labels.numel(), count, [&](auto block) {
      constexpr int BLOCK = decltype(block)::value;
      hipLaunchKernelGGL((sequence_coef_kernel<BLOCK>), dim3(count), dim3(BLOCK), 0, current_stream(), g,
                         labels.data_ptr<long>(), ignore, seqs, average, coef.data_ptr<float>());
    });
  HIP_CHECK(hipGetLastError());
  return coef;
}

// -> (loss, chosen rewards, rejected rewards, kept)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> preference_forward(
    const at::Tensor& logits, const at::Tensor& labels, const at::Tensor& ref, const c10::optional<at::Tensor>& cu,
    long pairs, long kind, double beta, double smoothing, bool average, long ignore) {
  check_rows(logits, labels);
  const at::DeviceGuard guard(logits.device());
  TORCH_CHECK(labels.numel() > 0 && pairs > 0, "preference_loss: needs a pair and a row");
  const Sequences seqs = sequences_of(labels, cu, 2 * pairs);
  const float* rf = floats(ref, logits, 2 * pairs, "ref_log_probs");
  const long rows = labels.numel();
  auto opts = logits.options().dtype(at::kFloat);
  const Kept kept = Kept::make(opts, rows, cu.has_value());
  auto chosen = at::empty({pairs}, opts), rejected = at::empty({pairs}, opts), loss = at::empty({}, opts);
  auto room = at::empty({rows + pairs + 1}, opts.dtype(at::kDouble));  // log-probabilities, the pairs' losses, the counter
  double *lp = room.data_ptr<double>(), *partial = lp + rows;
  int* arrived = (int*)(partial + pairs);
  launch_stats(logits, labels, ignore, 1.0, kept.stats, nullptr, lp, arrived);
  by_length(rows, 2 * pairs, [&](auto block) {
    constexpr int BLOCK = decltype(block)::value;
    hipLaunchKernelGGL((preference_kernel<BLOCK>), dim3(pairs), dim3(BLOCK), 0, current_stream(), lp,
                       labels.data_ptr<long>(), ignore, seqs, rf, pairs, (int)kind, beta, smoothing, average,
                       kept.coef, chosen.data_ptr<float>(), rejected.data_ptr<float>(), partial, arrived,
                       loss.data_ptr<float>());
  });
  HIP_CHECK(hipGetLastError());
  return {loss, chosen, rejected, kept.room};
}

// -> (loss, lp, kept)
std::tuple<at::Tensor, at::Tensor, at::Tensor> policy_forward(
    const at::Tensor& logits, const at::Tensor& labels, const c10::optional<at::Tensor>& old,
    const at::Tensor& advantages, bool by_row, const c10::optional<at::Tensor>& ref,
    const c10::optional<at::Tensor>& cu, long count, double low, double high, double kl, double temperature,
    long reduction, long ignore) {
  check_rows(logits, labels);
  const at::DeviceGuard guard(logits.device());
  const long rows = labels.numel();
  TORCH_CHECK(rows > 0 && count > 0, "policy_loss: needs a sequence and a row");
  const Sequences seqs = sequences_of(labels, cu, count);
  const Policy policy = policy_of(logits, old, advantages, by_row, ref, rows, count, low, high, kl);
  auto opts = logits.options().dtype(at::kFloat);
  const Kept kept = Kept::make(opts, rows, cu.has_value());
  auto lp = at::empty(labels.sizes(), opts);
  at::Tensor loss;
  if (reduction == NONE) loss = cu ? at::zeros(labels.sizes(), opts) : at::empty(labels.sizes(), opts);
  else loss = at::empty({}, opts);
  auto room = at::empty({2 * count + 1}, opts.dtype(at::kDouble));  // the sequences' losses and tokens, the counter
  double* partial = room.data_ptr<double>();
  int* arrived = (int*)(partial + 2 * count);
  launch_stats(logits, labels, ignore, temperature, kept.stats, lp.data_ptr<float>(), nullptr, arrived);
  by_length(rows, count, [&](auto block) {
    constexpr int BLOCK = decltype(block)::value;
    hipLaunchKernelGGL((policy_kernel<BLOCK>), dim3(count), dim3(BLOCK), 0, current_stream(), lp.data_ptr<float>(),
                       labels.data_ptr<long>(), ignore, seqs, policy, (int)reduction, kept.coef,
                       loss.data_ptr<float>(), partial, arrived, kept.norm, loss.data_ptr<float>());
  });
  HIP_CHECK(hipGetLastError());
  return {loss, lp, kept.room};
}

// The gradient is made here, for a gradient of the loss that is known -> (loss, lp, dlogits, applied)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> policy_at_once(
    at::Tensor logits, const at::Tensor& labels, const c10::optional<at::Tensor>& old, const at::Tensor& advantages,
    bool by_row, const c10::optional<at::Tensor>& ref, const c10::optional<at::Tensor>& cu, long count, double low,
    double high, double kl, double temperature, long reduction, long ignore, double scale,
    const c10::optional<at::Tensor>& scale_tensor) {
  check_rows(logits, labels);
  const at::DeviceGuard guard(logits.device());
  const long rows = labels.numel(), V = logits.size(-1);
  TORCH_CHECK(rows > 0 && count > 0, "policy_loss: needs a sequence and a row");
  TORCH_CHECK(reduction != NONE, "policy_loss: a gradient at once needs a loss of one number");
  auto opts = logits.options().dtype(at::kFloat);
  const Sequences seqs = sequences_of(labels, cu, count);
  const Policy policy = policy_of(logits, old, advantages, by_row, ref, rows, count, low, high, kl);
  const float* value = scale_tensor ? floats(*scale_tensor, logits, 1, "grad_scale") : nullptr;
  const long groups = reduction == SEQUENCE ? count : 1;
  const long blocks = std::min<long>(64, (rows + 4 * TOTAL_BLOCK - 1) / (4 * TOTAL_BLOCK));
  // blocks' sums in 64 bits, what the gradient is multiplied by, a counter, the weights, and the rows' losses
  auto room = at::empty({2 * blocks + 2 + groups + rows}, opts);
  auto* partial = (double*)room.data_ptr<float>();
  auto applied = room.narrow(0, 2 * blocks, 1);
  float *ap = (float*)(partial + blocks), *weights = ap + 2, *losses = weights + groups;
  int* arrived = (int*)(ap + 1);
  hipLaunchKernelGGL(policy_prepare_kernel, dim3(groups), dim3(PREPARE_BLOCK), 0, current_stream(),
                     labels.data_ptr<long>(), ignore, seqs, count, (int)reduction, (float)scale, value, ap, weights,
                     arrived);
  HIP_CHECK(hipGetLastError());
  at::Tensor grad, loss, lp;
  APEX_DISPATCH_FLOAT_HALF_BF(logits.scalar_type(), "policy_loss", ([&] {
    const long packs = V / Pack<scalar_t>::width;  // one less in rows at odd addresses
    auto launch = [&](auto block, auto most) {
      constexpr int BLOCK = decltype(block)::value, NP = decltype(most)::value;
      if (grad.defined() || packs > BLOCK * NP) return;
      grad = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
      loss = at::empty({}, opts);
      lp = at::empty(labels.sizes(), opts);
      const Rows where = rows_of(logits);
      constexpr long MOST = 1 << 20;  // a launch's threads are counted in 32 bits
      for (long first = 0; first < rows; first += MOST)
        hipLaunchKernelGGL((policy_at_once_kernel<scalar_t, BLOCK, NP>), dim3(std::min(MOST, rows - first)),
                           dim3(BLOCK), 0, current_stream(), (const scalar_t*)logits.data_ptr(), where,
                           labels.data_ptr<long>(), ignore, V, first, base_of(temperature), 1.0 / temperature, seqs,
                           count, policy, reduction == SEQUENCE, weights, ap, lp.data_ptr<float>(), losses,
                           (scalar_t*)grad.data_ptr());
    };
    auto launch_of = [&](auto block, auto... most) { (launch(block, most), ...); };
    // the fewest lanes that hold a row in up to 16 packs each: there is room for other rows on the compute unit then,
    // which read while this one waits for its sum
    using std::integral_constant;
    launch_of(integral_constant<int, 64>{}, integral_constant<int, 2>{}, integral_constant<int, 4>{},
              integral_constant<int, 6>{}, integral_constant<int, 8>{});
    launch_of(integral_constant<int, 256>{}, integral_constant<int, 4>{},
              integral_constant<int, 6>{}, integral_constant<int, 8>{}, integral_constant<int, 10>{},
              integral_constant<int, 12>{}, integral_constant<int, 14>{}, integral_constant<int, 16>{});
    launch_of(integral_constant<int, 512>{}, integral_constant<int, 10>{}, integral_constant<int, 12>{},
              integral_constant<int, 14>{}, integral_constant<int, 16>{});
    launch_of(integral_constant<int, 1024>{}, integral_constant<int, 10>{}, integral_constant<int, 12>{},
              integral_constant<int, 14>{}, integral_constant<int, 16>{});
  }()));
  HIP_CHECK(hipGetLastError());
  if (!grad.defined()) {  // a longer row is read twice
    auto [loss2, lp2, room2] = policy_forward(logits, labels, old, advantages, by_row, ref, cu, count, low, high, kl,
                                              temperature, reduction, ignore);
    const Kept kept = Kept::of(room2, rows);
    return {loss2, lp2, rows_backward(logits, labels, kept.stats, kept.coef, applied, kept.norm, ignore, temperature),
            applied};
  }
  hipLaunchKernelGGL(total_kernel, dim3(blocks), dim3(TOTAL_BLOCK), 0, current_stream(), losses, rows, partial, arrived,
                     loss.data_ptr<float>());
  HIP_CHECK(hipGetLastError());
  return {loss, lp, grad, applied};
}

void rescale_(at::Tensor grad, at::Tensor scale, at::Tensor applied) {
  const at::DeviceGuard guard(grad.device());
  TORCH_CHECK(grad.is_contiguous(), "rescale_: the gradient must be contiguous");
  const float *s = floats(scale, grad, 1, "grad_output"), *a = floats(applied, grad, 1, "applied");
  const long n = grad.numel();
  if (!n) return;
  const unsigned grid = (unsigned)std::min<long>((n + 2047) / 2048, 2048);
  APEX_DISPATCH_FLOAT_HALF_BF(grad.scalar_type(), "rescale_", ([&] {
    hipLaunchKernelGGL((rescale_kernel<scalar_t>), dim3(grid), dim3(256), 0, current_stream(),
                       (scalar_t*)grad.data_ptr(), n, s, a);
  }()));
  HIP_CHECK(hipGetLastError());
}

// ---------------- autograd ----------------
// In C++, so that the backward pass does not wait for the interpreter.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The gradient is not differentiable: said when it is differentiated, not when it is made.
at::Tensor once(const char* name, at::Tensor grad) {
  if (!at::GradMode::is_enabled()) return grad;
  grad.set_requires_grad(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " can be differentiated once only", 1);
  return (*error)({grad})[0];
}

// What is kept between the passes; `room` is a Kept's, or the rows' statistics alone
void keep(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& labels, const at::Tensor& room, long ignore,
          double temperature) {
  ctx->save_for_backward({logits, labels, room});
  ctx->saved_data["ignore"] = (int64_t)ignore;
  ctx->saved_data["temperature"] = temperature;
  ctx->set_materialize_grads(false);
}

at::Tensor fp32(const at::Tensor& t) { return t.to(at::kFloat).contiguous(); }

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& labels, int64_t ignore,
                            double temperature) {
    auto [lp, stats] = token_forward(logits, labels, ignore, temperature);
    keep(ctx, logits, labels, stats, ignore, temperature);
    return lp;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {{}, {}, {}, {}};
    const auto saved = ctx->get_saved_variables();
    const auto coef = fp32(grads[0].detach());
    auto grad = rows_backward(saved[0], saved[1], saved[2].data_ptr<float>(), floats(coef, saved[0], saved[1].numel(), "grad_output"),
                              {}, nullptr, ctx->saved_data["ignore"].toInt(), ctx->saved_data["temperature"].toDouble());
    return {once("token_log_probs", grad), {}, {}, {}};
  }
};

struct SequenceLogProbs : torch::autograd::Function<SequenceLogProbs> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& labels,
                            const c10::optional<at::Tensor>& cu, int64_t count, bool average, int64_t ignore,
                            double temperature) {
    auto [sums, stats] = sequence_forward(logits, labels, cu, count, average, ignore, temperature);
    keep(ctx, logits, labels, stats, ignore, temperature);
    ctx->save_for_backward({logits, labels, stats, cu ? *cu : at::Tensor()});
    ctx->saved_data["average"] = average;
    return sums;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {{}, {}, {}, {}, {}, {}, {}};
    const auto saved = ctx->get_saved_variables();
    const long ignore = ctx->saved_data["ignore"].toInt();
    const auto cu = saved[3].defined() ? c10::optional<at::Tensor>(saved[3]) : c10::nullopt;
    auto coef = sequence_coef(fp32(grads[0].detach()), saved[1], cu, ctx->saved_data["average"].toBool(), ignore);
    auto grad = rows_backward(saved[0], saved[1], saved[2].data_ptr<float>(), coef.data_ptr<float>(), {}, nullptr, ignore,
                              ctx->saved_data["temperature"].toDouble());
    return {once("sequence_log_probs", grad), {}, {}, {}, {}, {}, {}};
  }
};

// The backward pass of a loss whose coefficients the forward pass has made
at::Tensor loss_backward(const char* name, AutogradContext* ctx, const at::Tensor& given, bool with_norm) {
  const auto saved = ctx->get_saved_variables();
  const Kept kept = Kept::of(saved[2], saved[1].numel());
  return once(name, rows_backward(saved[0], saved[1], kept.stats, kept.coef, fp32(given.detach()),
                                  with_norm ? kept.norm : nullptr, ctx->saved_data["ignore"].toInt(),
                                  ctx->saved_data["temperature"].toDouble()));
}

struct PreferenceCall {
  at::Tensor labels, ref;
  c10::optional<at::Tensor> cu;
  long pairs, kind;
  double beta, smoothing;
  bool average;
  long ignore;
};

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const PreferenceCall& a) {
    auto [loss, chosen, rejected, room] = preference_forward(logits, a.labels, a.ref, a.cu, a.pairs, a.kind, a.beta,
                                                             a.smoothing, a.average, a.ignore);
    keep(ctx, logits, a.labels, room, a.ignore, 1.0);
    ctx->mark_non_differentiable({chosen, rejected});
    return {loss, chosen, rejected};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {{}, {}};
    return {loss_backward("preference_loss", ctx, grads[0], false), {}};
  }
};

struct PolicyCall {
  at::Tensor labels, advantages;
  c10::optional<at::Tensor> old, ref, cu, scale_tensor;
  bool by_row;
  long count, reduction, ignore;
  double low, high, kl, temperature, scale;
};

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const PolicyCall& a) {
    auto [loss, lp, room] = policy_forward(logits, a.labels, a.old, a.advantages, a.by_row, a.ref, a.cu, a.count, a.low,
                                           a.high, a.kl, a.temperature, a.reduction, a.ignore);
    keep(ctx, logits, a.labels, room, a.ignore, a.temperature);
    ctx->saved_data["norm"] = a.reduction == TOKEN;
    ctx->mark_non_differentiable({lp});
    return {loss, lp};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {{}, {}};
    return {loss_backward("policy_loss", ctx, grads[0], ctx->saved_data["norm"].toBool()), {}};
  }
};

// The loss and, in the same pass over the logits, their gradient for a gradient of the loss that is known
struct PolicyLossAtOnce : torch::autograd::Function<PolicyLossAtOnce> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const PolicyCall& a) {
    auto [loss, lp, grad, applied] = policy_at_once(logits, a.labels, a.old, a.advantages, a.by_row, a.ref, a.cu, a.count,
                                                    a.low, a.high, a.kl, a.temperature, a.reduction, a.ignore, a.scale,
                                                    a.scale_tensor);
    ctx->saved_data["grad"] = grad;
    ctx->saved_data["applied"] = applied;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({lp});
    return {loss, lp};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {{}, {}};
    TORCH_CHECK(ctx->saved_data.count("grad"),
                "policy_loss(grad_scale=...) made its gradient in the forward pass: it can be taken once only");
    auto grad = ctx->saved_data["grad"].toTensor();
    rescale_(grad, fp32(grads[0].detach()), ctx->saved_data["applied"].toTensor());
    ctx->saved_data.erase("grad");
    return {once("policy_loss", grad), {}};
  }
};

at::Tensor token_log_probs(at::Tensor logits, at::Tensor labels, long ignore, double temperature) {
  return TokenLogProbs::apply(logits, labels, (int64_t)ignore, temperature);
}

at::Tensor sequence_log_probs(at::Tensor logits, at::Tensor labels, c10::optional<at::Tensor> cu, long count,
                              bool average, long ignore, double temperature) {
  return SequenceLogProbs::apply(logits, labels, cu, (int64_t)count, average, (int64_t)ignore, temperature);
}

variable_list preference_loss(at::Tensor logits, at::Tensor labels, at::Tensor ref, c10::optional<at::Tensor> cu,
                              long pairs, long kind, double beta, double smoothing, bool average, long ignore) {
  return PreferenceLoss::apply(logits, PreferenceCall{labels, ref, cu, pairs, kind, beta, smoothing, average, ignore});
}

variable_list policy_loss(at::Tensor logits, at::Tensor labels, c10::optional<at::Tensor> old, at::Tensor advantages,
                          bool by_row, c10::optional<at::Tensor> ref, c10::optional<at::Tensor> cu, long count,
                          double low, double high, double kl, double temperature, long reduction, long ignore,
                          bool at_once, double scale, c10::optional<at::Tensor> scale_tensor) {
  const PolicyCall a{labels, advantages, old, ref, cu, scale_tensor, by_row, count, reduction, ignore,
                     low, high, kl, temperature, scale};
  // without a backward pass there is no gradient to make
  if (at_once && logits.requires_grad() && at::GradMode::is_enabled()) return PolicyLossAtOnce::apply(logits, a);
  return PolicyLoss::apply(logits, a);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("token_log_probs", &token_log_probs, "log-probabilities of given tokens");
  m.def("sequence_log_probs", &sequence_log_probs, "log-probabilities of sequences");
  m.def("preference_loss", &preference_loss, "paired log ratios -> (loss, chosen rewards, rejected rewards)");
  m.def("policy_loss", &policy_loss, "clipped policy loss with KL -> (loss, log-probabilities)");
}
