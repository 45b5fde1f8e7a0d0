// multi_tensor_adam_8bit — Adam/AdamW over many tensors with both moments in 8 bits.
//
// Mathematics. A moment is kept in blocks of 128 elements, in memory order from
// the tensor's start: one fp32 scale s = max|x| / 448 and codes q in e4m3 (OCP,
// 448 the largest), x = s q. The second moment v is kept as its root r, which
// halves the octaves that its values span (a block holds r down to 2^-17 of its
// largest). The step itself is in fp32 from the unrounded new moments.
//   m = b1 m + (1 - b1) g,  v = b2 r^2 + (1 - b2) g^2
//   p -= lr (m / bc1 / (sqrt(v) / sqrt(bc2) + eps) + wd p)
//
// Rounding. A step of b2 = 0.999 moves r by 0.05% a step where neighbouring codes
// are 6 to 12% apart: rounded to nearest, r would never move. So a value becomes
// the code below or above it at random, with odds that keep the mean of m, and of
// v (not of r): P(above) = (x - lo) / (hi - lo), and (r^2 - lo^2) / (hi^2 - lo^2).
// An r over 0 never becomes 0, for its inverse is used. The random numbers are a
// hash of (seed, step, tensor, element): 16 bits for m, 16 for v. A run repeats
// bit for bit, whatever the launch.
// A value that is not finite becomes the code NaN in its place alone: a block's
// scale is of its finite values.
//
// What bounds it: HBM. Per element of fp32 weights 12 B (g, p in and out) + 4 B
// of moments + 0.125 B of scales, against 28 B with fp32 moments. 682M bf16
// weights with masters (16.1 B each): 1.89 ms, 5.8 TB/s; 216M fp32 0.60 ms.
#include "amp_C.h"
#include "multi_tensor_apply.h"

#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <cmath>

namespace {

// Each lane has four neighbouring elements and is done: every load and store of a
// wave is one piece without gaps, whatever the type, and may go past the caches.
// With eight a lane (two loads of 16 bytes, 32 apart, for fp32) the same took 4% and
// 8% longer; workgroups that went on to a second to eighth part 5 to 15%, for nothing
// was on its way while they rounded. 682M bf16 weights with masters and 216M fp32
// weights take 1875 and 600 us by 256 threads, 1895 and 604 by 128, 1975 and 625 by
// 512, 2045 and 655 by 1024.
constexpr int A8_BLOCK = 256;          // threads
constexpr int A8_PER_LANE = 4;         // elements: 32 lanes have a block of 128
constexpr int A8_SCALE_BLOCK = 128;    // elements of one scale
constexpr int A8_CHUNK = A8_BLOCK * A8_PER_LANE;  // elements of a workgroup
constexpr int A8_TENSORS = 48;         // of one launch: 48 * 72 B of kernel arguments
constexpr long A8_SIDE = 1 << 23;      // workgroups along a grid's x
constexpr float E4M3_MAX = 448.f;

struct Adam8Meta {
  void* g[A8_TENSORS];
  void* p[A8_TENSORS];
  void* master[A8_TENSORS];
  unsigned char* m[A8_TENSORS];
  unsigned char* r[A8_TENSORS];
  float* m_scale[A8_TENSORS];
  float* r_scale[A8_TENSORS];
  long sizes[A8_TENSORS];
  int ordinal[A8_TENSORS];           // of the tensor in the optimizer, for its random numbers
  int chunk_prefix[A8_TENSORS + 1];  // cumulative chunks
  int ntensors;
};

struct Adam8Args {
  double beta1_d, beta2_d;
  float lr, beta1, beta2, rest1, rest2;  // rest = 1 - beta, of the 64-bit beta: in 32 bits 1 - 0.999 is 1e-5 off
  float eps, bc1_recip, bc2_root_recip, decay;
  int mode, bias_correction;
  unsigned seed;
  int step;
  // capturable: read on the device at every replay
  const float *lr_ptr, *inv_scale, *found_inf;
  const int* step_ptr;
};

// Multiply-xorshift mixing of 32 bits; the odd multipliers are the largest prime up
// to 2^32 over the golden ratio, and the leading fractional bits of the root of 3.
__device__ __forceinline__ unsigned mix32(unsigned x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}

// The largest of a block's 32 lanes, on each of them: exchanges within quads,
// mirrored halves and rows of 16, then between two rows. None needs LDS.
__device__ __forceinline__ float max32(float v) {
#define A8_DPP(ctrl) \
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), ctrl, 0xF, 0xF, true)))
  A8_DPP(0xB1);   // quad_perm 1,0,3,2
  A8_DPP(0x4E);   // quad_perm 2,3,0,1
  A8_DPP(0x141);  // row_half_mirror
  A8_DPP(0x140);  // row_mirror
#undef A8_DPP
  const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  return fmaxf(__int_as_float(rows[0]), __int_as_float(rows[1]));
}

// A |y| <= 448 lies between two neighbouring codes; u = (b + 0.5) / 65536 chooses.
// 448 is a code: a maximum that is one rounding over it has odds under any u.
// fma(|y|, 0, q) is q, without the sign of a -0, and NaN where y is not finite.

// The first moment: up where u < z - k, z = k + rest the value in codes. In the
// float's bits the rest is the lower 20, and the condition that rest + 2^20 -
// (16 b + 9) carries. Under 2^-6 codes are evenly 2^-9 apart, as they are from
// 2^-6 to 2^-5: the value is moved there and back.
__device__ __forceinline__ float choose_linear(float y, unsigned b) {
  const float move = fabsf(y) < 0.015625f ? 0.015625f : 0.f;
  const unsigned carry = ((~b & 0xFFFFu) << 4) | 7u;
  const unsigned q = (__float_as_uint(fabsf(y) + move) + carry) & 0xFFF00000u;
  return fmaf(fabsf(y), 0.f, copysignf(__uint_as_float(q) - move, y));
}

// The root: up where u < (z^2 - k^2) / ((k + 1)^2 - k^2), and always from 0.
__device__ __forceinline__ float choose_root(float y, unsigned b) {
  const float u = ((float)b + 0.5f) * (1.f / 65536.f);
  // step = 2^(exponent - 3), not under 2^-9
  const int step_bits = max(__float_as_int(y) & 0x7F800000, 121 << 23) - (3 << 23);
  const float step = __int_as_float(step_bits), inv = __int_as_float((254 << 23) - step_bits);
  const float z = y * inv, k = floorf(z);
  const float n = u * fmaf(2.f, k, 1.f) < (z - k) * (z + k) ? k + 1.f : k;
  return fmaf(y, 0.f, fmaxf(n, y > 0.f ? 1.f : n) * step);
}

// sqrtf but for one operand in some thousands (its last bit), in half the
// instructions: the hardware's root (1 ulp) and one Newton step from its residual.
// The hardware takes a subnormal for 0, and infinity's residual is NaN: sqrtf has
// them, in a branch that hardly any wave takes. 682M bf16 weights with masters take
// 1892 us so, 1888 without the branch, 1911 with one for each element, 1936 by sqrtf.
constexpr int FAR = 0x080 | 0x200;  // v_cmp_class: positive subnormal, positive infinity
__device__ __forceinline__ void roots(float (&v)[4]) {
  float r[4];
  bool far = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float near = __builtin_amdgcn_sqrtf(v[j]);
    const float half = 0.5f * __builtin_amdgcn_rcpf(fmaxf(near, 1e-30f));
    r[j] = fmaf(fmaf(-near, near, v[j]), half, near);
    far = far || __builtin_amdgcn_classf(v[j], FAR);
  }
  if (__any(far)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = sqrtf(v[j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = r[j];
}

typedef float float2v __attribute__((ext_vector_type(2)));

template <typename T>
struct Four {
  T a[4];
};

// Four elements at an address that is aligned to its element only (views into one
// buffer), past the caches: a step meets each once.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_at_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2_at_2 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned u32_at_1 __attribute__((aligned(1)));

template <typename T>
__device__ __forceinline__ Four<T> load4(const T* p) {
  Four<T> v;
  if constexpr (sizeof(T) == 4) {
    const u32x4 w = __builtin_nontemporal_load((const u32x4_at_4*)p);
    __builtin_memcpy(&v, &w, 16);
  } else if constexpr (sizeof(T) == 2) {
    const u32x2 w = __builtin_nontemporal_load((const u32x2_at_2*)p);
    __builtin_memcpy(&v, &w, 8);
  } else {
    const unsigned w = __builtin_nontemporal_load((const u32_at_1*)p);
    __builtin_memcpy(&v, &w, 4);
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const Four<T>& v) {
  if constexpr (sizeof(T) == 4) {
    u32x4 w;
    __builtin_memcpy(&w, &v, 16);
    __builtin_nontemporal_store(w, (u32x4_at_4*)p);
  } else if constexpr (sizeof(T) == 2) {
    u32x2 w;
    __builtin_memcpy(&w, &v, 8);
    __builtin_nontemporal_store(w, (u32x2_at_2*)p);
  } else {
    unsigned w;
    __builtin_memcpy(&w, &v, 4);
    __builtin_nontemporal_store(w, (u32_at_1*)p);
  }
}

__device__ __forceinline__ void decode4(const Four<unsigned char>& c, float* x) {
  int w;
  __builtin_memcpy(&w, &c, 4);
  const float2v lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  x[0] = lo.x;
  x[1] = lo.y;
  x[2] = hi.x;
  x[3] = hi.y;
}

__device__ __forceinline__ Four<unsigned char> encode4(const float* q) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
  Four<unsigned char> c;
  __builtin_memcpy(&c, &w, 4);
  return c;
}

// Scale and codes of a lane's four values, with its block's other 31 lanes.
template <bool ROOT>
__device__ __forceinline__ float encode_block(const float* x, const unsigned* bits, Four<unsigned char>& codes) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(x[j]));  // NaN is no part of it
  top = max32(top);
  if (__any(top == INFINITY)) {  // nor is infinity: hardly ever met
    top = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fabsf(x[j]) < INFINITY ? fmaxf(top, fabsf(x[j])) : top;
    top = max32(top);
  }
  const float scale = fmaxf(top * (1.f / E4M3_MAX), 1.17549435e-38f), inv = 1.f / scale;
  float q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    q[j] = ROOT ? choose_root(x[j] * inv, bits[j] >> 16) : choose_linear(x[j] * inv, bits[j] & 0xFFFFu);
  codes = encode4(q);
  return scale;
}

// The new moments, each product and sum rounded by itself, as elementary operations
// do it: a code or scale that fell to the other side by a last bit would show in
// all that follows. (The _rn functions are plain products and sums to the compiler,
// which fuses them.)
__device__ __forceinline__ float mean_of(float beta, float m, float rest, float g) {
#pragma clang fp contract(off)
  const float old = beta * m, now = rest * g;
  return old + now;
}
__device__ __forceinline__ float square_of(float beta, float r, float rest, float g) {
#pragma clang fp contract(off)
  const float old = beta * r * r, now = rest * g * g;
  return old + now;
}

template <typename T, bool MASTER>
__global__ void __launch_bounds__(A8_BLOCK) adam_8bit_kernel(Adam8Meta meta, Adam8Args a) {
  __shared__ float corrections[2];
  if (a.found_inf && *a.found_inf != 0.f) return;
  int step = a.step;
  if (a.step_ptr) {
    step = *a.step_ptr;
    if (threadIdx.x == 0) {
      corrections[0] = a.bias_correction ? (float)(1.0 / (1.0 - pow(a.beta1_d, (double)step))) : 1.f;
      corrections[1] = a.bias_correction ? (float)(1.0 / sqrt(1.0 - pow(a.beta2_d, (double)step))) : 1.f;
    }
    __syncthreads();
    a.bc1_recip = corrections[0];
    a.bc2_root_recip = corrections[1];
  }
  if (a.lr_ptr) a.lr = *a.lr_ptr;
  const float unscale = a.inv_scale ? *a.inv_scale : 1.f;

  // a grid counts threads in 32 bits along each side: the chunks of more than 2^33 elements go on along y, and the last
  // row of workgroups may lie behind the last tensor, where no lane has an element
  const int chunk = (int)(blockIdx.y * gridDim.x + blockIdx.x);
  int t = 0;
  {
    int hi = meta.ntensors - 1;
    while (t < hi) {
      const int mid = (t + hi + 1) >> 1;
      if (meta.chunk_prefix[mid] <= chunk) t = mid; else hi = mid - 1;
    }
  }
  const long n = meta.sizes[t], base = (long)(chunk - meta.chunk_prefix[t]) * A8_CHUNK;
  T* gp = (T*)meta.g[t];
  T* pp = (T*)meta.p[t];
  float* wp = (float*)meta.master[t];
  const unsigned key = mix32(a.seed ^ mix32((unsigned)step + mix32((unsigned)meta.ordinal[t] + 0x6A09E667u)));

  // lanes behind the tensor's end stay: a block's lanes exchange their maxima
  const long i = base + threadIdx.x * A8_PER_LANE;
  const int have = (int)min(max(n - i, 0L), 4L);
  float g[4], p[4], m[4], r[4];
  float sm = 0.f, sr = 0.f;
  if (have) {
    sm = meta.m_scale[t][i / A8_SCALE_BLOCK];
    sr = meta.r_scale[t][i / A8_SCALE_BLOCK];
  }
  if (have == 4) {
    const Four<T> vg = load4(gp + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = to_float(vg.a[j]);
    if (MASTER) {
      const Four<float> vw = load4(wp + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = vw.a[j];
    } else {
      const Four<T> vp = load4(pp + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = to_float(vp.a[j]);
    }
    decode4(load4(meta.m[t] + i), m);
    decode4(load4(meta.r[t] + i), r);
  } else {
    Four<unsigned char> cm, cr;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      g[j] = j < have ? to_float(gp[i + j]) : 0.f;
      p[j] = j < have ? (MASTER ? wp[i + j] : to_float(pp[i + j])) : 0.f;
      cm.a[j] = j < have ? meta.m[t][i + j] : 0;
      cr.a[j] = j < have ? meta.r[t][i + j] : 0;
    }
    decode4(cm, m);
    decode4(cr, r);
  }

  if (a.inv_scale) {
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] *= unscale;
  }
  if (a.mode == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = fmaf(a.decay, p[j], g[j]);
  }
  unsigned bits[4];
  float update[4];
  const unsigned high = (unsigned)(i >> 32) * 0x6A09E667u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bits[j] = mix32(((unsigned)i + j) * 0x9E3779B1u + key + high);
    m[j] = mean_of(a.beta1, m[j] * sm, a.rest1, g[j]);
    r[j] = square_of(a.beta2, r[j] * sr, a.rest2, g[j]);
  }
  roots(r);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    update[j] = (m[j] * a.bc1_recip) * __builtin_amdgcn_rcpf(fmaf(r[j], a.bc2_root_recip, a.eps));
  if (a.mode == 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) update[j] = fmaf(a.decay, p[j], update[j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    p[j] = fmaf(-a.lr, update[j], p[j]);
    // the param is the stored master's rounding: not that of an fma that rounds to fp16 at once
    if (MASTER) asm volatile("" : "+v"(p[j]));
  }
  if (have != 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j >= have) m[j] = r[j] = 0.f;
  }

  Four<unsigned char> cm, cr;
  const float new_sm = encode_block<false>(m, bits, cm);
  const float new_sr = encode_block<true>(r, bits, cr);
  if (have == 4) {
    if (MASTER) {
      Four<float> vw;
#pragma unroll
      for (int j = 0; j < 4; ++j) vw.a[j] = p[j];
      store4(wp + i, vw);
    }
    Four<T> vp;
#pragma unroll
    for (int j = 0; j < 4; ++j) vp.a[j] = from_float<T>(p[j]);
    store4(pp + i, vp);
    store4(meta.m[t] + i, cm);
    store4(meta.r[t] + i, cr);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < have) {
        if (MASTER) wp[i + j] = p[j];
        pp[i + j] = from_float<T>(p[j]);
        meta.m[t][i + j] = cm.a[j];
        meta.r[t][i + j] = cr.a[j];
      }
    }
  }
  if (have && i % A8_SCALE_BLOCK == 0) {
    meta.m_scale[t][i / A8_SCALE_BLOCK] = new_sm;
    meta.r_scale[t][i / A8_SCALE_BLOCK] = new_sr;
  }
}

Adam8Args args_of(double beta1, double beta2, double eps, long mode, long bias_correction, double decay, long seed) {
  Adam8Args a{};
  a.beta1_d = beta1;
  a.beta2_d = beta2;
  a.beta1 = (float)beta1;
  a.beta2 = (float)beta2;
  a.rest1 = (float)(1.0 - beta1);
  a.rest2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.decay = (float)decay;
  a.mode = (int)mode;
  a.bias_correction = (int)bias_correction;
  a.seed = (unsigned)seed;
  return a;
}

// tensor_lists: g, p, exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale(, master)
void adam_8bit(TensorLists& lists, const std::vector<long>& ordinals, const Adam8Args& args) {
  TORCH_CHECK(lists.size() == 6 || lists.size() == 7, "multi_tensor_adam_8bit: 6 lists, or 7 with master weights");
  const size_t count = lists[0].size();
  const bool master = lists.size() == 7;
  for (auto& l : lists) TORCH_CHECK(l.size() == count, "multi_tensor_adam_8bit: tensor list length mismatch");
  TORCH_CHECK(ordinals.size() == count, "multi_tensor_adam_8bit: one ordinal a tensor");
  if (!count) return;
  const auto device = lists[0][0].device();
  const auto type = lists[1][0].scalar_type();
  const at::DeviceGuard guard(device);
  auto stream = current_stream();
  // all are looked at before the first launch: a step that is refused has changed no tensor
  for (size_t t = 0; t < count; ++t) {
    // a gradient of another layout is met in the param's order; the copy lives until the launches are under way
    if (lists[0][t].strides() != lists[1][t].strides() && lists[0][t].numel() > 1)
      lists[0][t] = at::empty_like(lists[1][t]).copy_(lists[0][t]);
    const long n = lists[1][t].numel(), blocks = (n + A8_SCALE_BLOCK - 1) / A8_SCALE_BLOCK;
    for (size_t d = 0; d < lists.size(); ++d) {
      const auto& x = lists[d][t];
      const bool scales = d == 3 || d == 5;
      TORCH_CHECK(x.device() == device, "multi_tensor_adam_8bit: tensors on more than one device");
      TORCH_CHECK(x.numel() == (scales ? blocks : n), "multi_tensor_adam_8bit: size mismatch within tuple");
      TORCH_CHECK(x.is_non_overlapping_and_dense(), "multi_tensor_adam_8bit: tensor not dense/contiguous");
      TORCH_CHECK(scales || n <= 1 || x.strides() == lists[1][t].strides(),
                  "multi_tensor_adam_8bit: layout mismatch within tensor tuple");
      const auto want = d <= 1 ? type : d == 2 || d == 4 ? at::kFloat8_e4m3fn : at::kFloat;
      TORCH_CHECK(x.scalar_type() == want, "multi_tensor_adam_8bit: list ", d, " must be ", want, ", got ", x.scalar_type());
    }
  }
  Adam8Meta meta;
  size_t t = 0;
  while (t < count) {
    int nt = 0;
    long chunks = 0;
    while (t < count && nt < A8_TENSORS) {
      const long n = lists[1][t].numel();
      if (n) {
        meta.g[nt] = lists[0][t].data_ptr();
        meta.p[nt] = lists[1][t].data_ptr();
        meta.m[nt] = (unsigned char*)lists[2][t].data_ptr();
        meta.m_scale[nt] = lists[3][t].data_ptr<float>();
        meta.r[nt] = (unsigned char*)lists[4][t].data_ptr();
        meta.r_scale[nt] = lists[5][t].data_ptr<float>();
        meta.master[nt] = master ? lists[6][t].data_ptr() : nullptr;
        meta.sizes[nt] = n;
        meta.ordinal[nt] = (int)ordinals[t];
        meta.chunk_prefix[nt] = (int)chunks;
        chunks += (n + A8_CHUNK - 1) / A8_CHUNK;
        ++nt;
      }
      ++t;
    }
    if (!nt) continue;
    meta.chunk_prefix[nt] = (int)chunks;
    meta.ntensors = nt;
    const dim3 grid((unsigned)std::min(chunks, A8_SIDE), (unsigned)((chunks + A8_SIDE - 1) / A8_SIDE));
    APEX_DISPATCH_FLOAT_HALF_BF(type, "multi_tensor_adam_8bit", ([&] {
      if (master) {
        hipLaunchKernelGGL((adam_8bit_kernel<scalar_t, true>), grid, dim3(A8_BLOCK), 0, stream, meta, args);
      } else {
        hipLaunchKernelGGL((adam_8bit_kernel<scalar_t, false>), grid, dim3(A8_BLOCK), 0, stream, meta, args);
      }
    }()));
    HIP_CHECK(hipGetLastError());
  }
}

}  // namespace

void multi_tensor_adam_8bit_cuda(TensorLists tensor_lists, std::vector<long> ordinals, double lr, double beta1,
                                 double beta2, double eps, long step, long mode, long bias_correction,
                                 double weight_decay, long seed) {
  Adam8Args a = args_of(beta1, beta2, eps, mode, bias_correction, weight_decay, seed);
  a.lr = (float)lr;
  a.bc1_recip = bias_correction ? (float)(1.0 / (1.0 - std::pow(beta1, (double)step))) : 1.f;
  a.bc2_root_recip = bias_correction ? (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step))) : 1.f;
  a.step = (int)step;
  adam_8bit(tensor_lists, ordinals, a);
}

void multi_tensor_adam_8bit_capturable_cuda(TensorLists tensor_lists, std::vector<long> ordinals, at::Tensor lr,
                                            double beta1, double beta2, double eps, at::Tensor step, long mode,
                                            long bias_correction, double weight_decay, long seed,
                                            c10::optional<at::Tensor> inv_scale, c10::optional<at::Tensor> found_inf) {
  if (tensor_lists.empty() || tensor_lists[0].empty()) return;
  const auto device = tensor_lists[0][0].device();
  auto value = [&](const at::Tensor& t, at::ScalarType type, const char* name) {
    TORCH_CHECK(t.device() == device && t.numel() == 1 && t.scalar_type() == type, "multi_tensor_adam_8bit: ", name,
                " must be one ", type, " on the params' device");
    return t.data_ptr();
  };
  Adam8Args a = args_of(beta1, beta2, eps, mode, bias_correction, weight_decay, seed);
  a.lr_ptr = (const float*)value(lr, at::kFloat, "lr");
  a.step_ptr = (const int*)value(step, at::kInt, "step");
  if (inv_scale) a.inv_scale = (const float*)value(*inv_scale, at::kFloat, "inv_scale");
  if (found_inf) a.found_inf = (const float*)value(*found_inf, at::kFloat, "found_inf");
  adam_8bit(tensor_lists, ordinals, a);
}
