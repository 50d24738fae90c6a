// Root-mean-square norm that opens a block: the residual's addition in front of it, 16 / 32-bit or e4m3 output behind it
// (fla/modules/layernorm.py: rms_norm, RMSNorm; the 8-bit output is this library's own).
//   forward :  s = round(x + r);  y = s rstd w,  rstd = 1 / sqrt(mean(s^2) + eps);  8 bits: q = e4m3(y / scale), scale = max|y| / 448
//   backward:  xhat = s rstd;  ds = rstd (w dy - xhat mean(xhat w dy)) + ds_out;  dx = dr = ds;  dw = sum over rows of dy xhat
// s is the residual stream as it is stored (the type the caller keeps it in), and y is computed from that stored value: the same
// numbers as the unfused pair, and backward, which reads s, differentiates exactly what forward computed.  Everything else is fp32,
// rounded once when stored.
//
// Bound by HBM: every element is read and written once.  A row belongs to TPR threads (32 to 512) that keep it in registers, NV
// vectors of 16 bytes each; rows whose length or address does not allow vectors go element by element, and rows too long for
// that are read again from L2 (NV = 0).  dw: every thread sums its columns over the rows of its block in registers, one partial row a
// block, and a second small kernel adds the partial rows in order: no atomics, results repeat bit for bit.
#include <cuda_fp8.h>

#include <initializer_list>

#include "common.cuh"

namespace flab {
namespace {

constexpr float E4M3_MAX = 448.f;

struct NormParams {
  const void *x, *res, *w;
  void *y, *sum;
  float *rstd, *scale;
  long long rows;
  int n, tpr;
  int res_fp32, w_type;
  float eps;
};

template <typename T, int V> struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Vec {
  T v[V];
};

template <typename T, int V> __device__ __forceinline__ void load_f(const void *base, size_t at, float (&f)[V]) {
  const Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(reinterpret_cast<const T *>(base) + at);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = Num<T>::f(v.v[j]);
}
template <typename T, int V> __device__ __forceinline__ void store_f(void *base, size_t at, const float (&f)[V]) {
  Vec<T, V> v;
#pragma unroll
  for (int j = 0; j < V; ++j) v.v[j] = Num<T>::t(f[j]);
  *reinterpret_cast<Vec<T, V> *>(reinterpret_cast<T *>(base) + at) = v;
}
// the weight has a type of its own
template <int V> __device__ __forceinline__ void load_w(const void *w, int type, int at, float (&f)[V]) {
  if (!w) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = 1.f;
  } else if (type == FLAB_BF16) {
    load_f<bf16, V>(w, at, f);
  } else if (type == FLAB_FP16) {
    load_f<__half, V>(w, at, f);
  } else {
    load_f<float, V>(w, at, f);
  }
}

// sum (or maximum, where a NaN wins) over the TPR threads of a row; `slot` is a row of shared memory per warp of the block
template <bool MAX> __device__ __forceinline__ float join(float a, float b) { return MAX ? (b > a || b != b ? b : a) : a + b; }
template <bool MAX> __device__ __forceinline__ float row_reduce(float v, int tpr, float *slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join<MAX>(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5, first = threadIdx.x / tpr * (tpr >> 5);
    if ((threadIdx.x & 31) == 0) slot[warp] = v;
    __syncthreads();
    v = slot[first];
    for (int i = 1; i < tpr >> 5; ++i) v = join<MAX>(v, slot[first + i]);
  }
  return v;
}

// V e4m3 bytes, values beyond the type's range held at its largest (a NaN stays one)
template <int V> __device__ __forceinline__ void store_e4m3(void *base, size_t at, const float (&f)[V], float inv) {
  Vec<unsigned char, V> q;
  if constexpr (V == 1) {
    q.v[0] = __nv_cvt_float_to_fp8(f[0] * inv, __NV_SATFINITE, __NV_E4M3);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(f[j] * inv, f[j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
      q.v[j] = two & 0xff, q.v[j + 1] = two >> 8;
    }
  }
  *reinterpret_cast<Vec<unsigned char, V> *>(reinterpret_cast<unsigned char *>(base) + at) = q;
}

// T: x and y;  S: the stored sum;  V elements a vector, NV vectors a thread (0: read again);  QUANT: e4m3 output;  NORM: without
// it the rows are quantised as they are
template <typename T, typename S, int V, int NV, bool QUANT, bool NORM>
__global__ void __launch_bounds__(NV ? 512 : 1024) rms_norm_fwd_kernel(const NormParams p) {
  __shared__ float slots[2][32];
  const int li = threadIdx.x % p.tpr;
  const long long row = (long long)blockIdx.x * (blockDim.x / p.tpr) + threadIdx.x / p.tpr;
  const bool on = row < p.rows;
  const size_t base = (size_t)row * p.n;
  constexpr int KEEP = NV ? NV : 1;
  const int loops = NV ? NV : (p.n + V * p.tpr - 1) / (V * p.tpr);
  float f[KEEP][V];

  auto fetch = [&](int c, float (&v)[V], bool first) {  // the stored sum of a vector
    load_f<T, V>(p.x, base + c, v);
    if (p.res) {
      float r[V];
      if (p.res_fp32) load_f<float, V>(p.res, base + c, r);
      else load_f<T, V>(p.res, base + c, r);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += r[j];
    }
    if (p.sum && first) store_f<S, V>(p.sum, base + c, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = rnd<S>(v[j]);
  };

  float ss = 0.f;
  if (on && (NORM || NV)) {
#pragma unroll
    for (int k = 0; k < (NV ? NV : loops); ++k) {
      const int c = (k * p.tpr + li) * V;
      float(&v)[V] = f[NV ? k : 0];
      if (c < p.n) {
        fetch(c, v, true);
#pragma unroll
        for (int j = 0; j < V; ++j) ss = fmaf(v[j], v[j], ss);
      }
    }
  }
  float rstd = 1.f;
  if (NORM) {
    ss = row_reduce<false>(ss, p.tpr, slots[0]);
    rstd = 1.f / sqrtf(ss / p.n + p.eps);
    if (on && li == 0 && p.rstd) p.rstd[row] = rstd;
  }
  float inv = 0.f;
  if (QUANT) {
    float top = 0.f;
    if (on) {
#pragma unroll
      for (int k = 0; k < (NV ? NV : loops); ++k) {
        const int c = (k * p.tpr + li) * V;
        float(&v)[V] = f[NV ? k : 0];
        if (c < p.n) {
          if (!NV) fetch(c, v, !NORM);
          float w[V];
          load_w<V>(p.w, p.w_type, c, w);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float y = v[j] * rstd * w[j];
            if (NV) v[j] = y;
            top = join<true>(top, fabsf(y));
          }
        }
      }
    }
    top = row_reduce<true>(top, p.tpr, slots[1]);
    // a row of zeros has scale 0 and zeros; a scale below what has a reciprocal is held there
    inv = top > 0.f ? fminf(E4M3_MAX / top, 3.4e38f) : top;
    if (on && li == 0) p.scale[row] = top / E4M3_MAX;
  }
  if (!on) return;
#pragma unroll
  for (int k = 0; k < (NV ? NV : loops); ++k) {
    const int c = (k * p.tpr + li) * V;
    float(&v)[V] = f[NV ? k : 0];
    if (c < p.n) {
      if (!NV) fetch(c, v, false);
      if (!(QUANT && NV)) {
        float w[V];
        load_w<V>(p.w, p.w_type, c, w);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = v[j] * rstd * w[j];
      }
      if constexpr (QUANT) store_e4m3<V>(p.y, base + c, v, inv);
      else store_f<T, V>(p.y, base + c, v);
    }
  }
}

struct NormBwdParams {
  const void *s, *dy, *ds, *w;
  const float *rstd;
  void *dx, *dr;
  float *part;
  long long rows;
  int n, tpr, w_type;
};

// one partial row of dw a block; the block's groups of TPR threads take rows in turn
template <typename T, typename S, int V, int NV> __global__ void __launch_bounds__(NV ? 256 : 1024) rms_norm_bwd_kernel(const NormBwdParams p) {
  extern __shared__ float sdw[];  // [groups][n]
  __shared__ float slots[2][32];
  const int li = threadIdx.x % p.tpr, group = threadIdx.x / p.tpr, groups = blockDim.x / p.tpr;
  constexpr int KEEP = NV ? NV : 1;
  const int loops = NV ? NV : (p.n + V * p.tpr - 1) / (V * p.tpr);
  float acc[KEEP][V] = {};
  if (!NV && p.part) {  // rows too long for registers: the thread's columns are its own in shared memory
    for (int k = 0; k < loops; ++k)
      for (int j = 0; j < V; ++j)
        if ((k * p.tpr + li) * V < p.n) sdw[(k * p.tpr + li) * V + j] = 0.f;
  }
  int par = 0;
  for (long long r0 = (long long)blockIdx.x * groups; r0 < p.rows; r0 += (long long)gridDim.x * groups, par ^= 1) {
    const long long row = r0 + group;
    const bool on = row < p.rows;
    const size_t base = (size_t)row * p.n;
    const float rstd = on ? p.rstd[row] : 0.f;
    float xh[KEEP][V], wd[KEEP][V], dot = 0.f;
    Vec<S, V> keep[KEEP];  // ds_out, asked for with the rest
    if (on) {
#pragma unroll
      for (int k = 0; k < (NV ? NV : loops); ++k) {
        const int c = (k * p.tpr + li) * V, i = NV ? k : 0;
        if (c < p.n) {
          float w[V], s[V], dy[V];
          load_f<S, V>(p.s, base + c, s);
          load_f<T, V>(p.dy, base + c, dy);
          if (NV && p.ds) keep[i] = *reinterpret_cast<const Vec<S, V> *>(reinterpret_cast<const S *>(p.ds) + base + c);
          load_w<V>(p.w, p.w_type, c, w);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            xh[i][j] = s[j] * rstd;
            wd[i][j] = w[j] * dy[j];
            dot = fmaf(xh[i][j], wd[i][j], dot);
            if (NV) acc[i][j] = fmaf(dy[j], xh[i][j], acc[i][j]);
            else if (p.part) sdw[c + j] = fmaf(dy[j], xh[i][j], sdw[c + j]);
          }
        }
      }
    }
    dot = row_reduce<false>(dot, p.tpr, slots[par]) / p.n;
    if (on) {
#pragma unroll
      for (int k = 0; k < (NV ? NV : loops); ++k) {
        const int c = (k * p.tpr + li) * V, i = NV ? k : 0;
        if (c < p.n) {
          if (!NV) {
            float w[V], s[V], dy[V];
            load_f<S, V>(p.s, base + c, s);
            load_f<T, V>(p.dy, base + c, dy);
            load_w<V>(p.w, p.w_type, c, w);
            if (p.ds) keep[i] = *reinterpret_cast<const Vec<S, V> *>(reinterpret_cast<const S *>(p.ds) + base + c);
#pragma unroll
            for (int j = 0; j < V; ++j) xh[i][j] = s[j] * rstd, wd[i][j] = w[j] * dy[j];
          }
          float d[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            d[j] = (wd[i][j] - xh[i][j] * dot) * rstd;
            if (p.ds) d[j] += Num<S>::f(keep[i].v[j]);
          }
          if (p.dx) store_f<T, V>(p.dx, base + c, d);
          if (p.dr) store_f<S, V>(p.dr, base + c, d);
        }
      }
    }
  }
  if (!p.part) return;
  if (NV) {
    for (int k = 0; k < (NV ? NV : 0); ++k) {
      const int c = (k * p.tpr + li) * V;
      if (c < p.n)
        for (int j = 0; j < V; ++j) sdw[(size_t)group * p.n + c + j] = acc[NV ? k : 0][j];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.n; c += blockDim.x) {
    float t = 0.f;
    for (int i = 0; i < groups; ++i) t += sdw[(size_t)i * p.n + c];
    p.part[(size_t)blockIdx.x * p.n + c] = t;
  }
}

// out[c] = sum over the partial rows, in order: 8 warps take every eighth row of 32 columns
template <typename T> __global__ void __launch_bounds__(256) partial_sum_kernel(const float *__restrict__ part, T *__restrict__ out, int parts, int n) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int i = w; i < parts; i += 8) t += part[(size_t)i * n + c];
  }
  s[w][lane] = t;
  __syncthreads();
  if (w == 0 && c < n) {
#pragma unroll
    for (int i = 1; i < 8; ++i) t += s[i][lane];
    out[c] = Num<T>::t(t);
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Threads a row and vectors a thread for `groups` vectors a row: the fewest threads that hold the row in `most` vectors each, then
// more of them while the rows alone do not fill the card (512 threads an SM).
void norm_split(long long rows, long long groups, int most, int &tpr, int &nv) {
  tpr = 32;
  while (tpr < 512 && groups > (long long)tpr * most) tpr *= 2;
  const long long fill = (long long)sm_count() * 512;
  while (tpr < 256 && groups > tpr && rows * tpr < fill) tpr *= 2;
  const long long need = (groups + tpr - 1) / tpr;
  nv = need > most ? 0 : need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : need <= 8 ? 8 : 16;
  if (nv == 0) tpr = 1024;
}

bool aligned16(std::initializer_list<const void *> ptrs) {
  for (const void *q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return false;
  return true;
}

template <typename T, typename S, bool QUANT, bool NORM> int launch_norm_fwd(NormParams p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = p.n % V == 0 && aligned16({p.x, p.res, p.w, p.y, p.sum});
  int nv;
  norm_split(p.rows, vec ? p.n / V : p.n, 8, p.tpr, nv);
  const int block = p.tpr < 128 ? 128 : p.tpr;
  const unsigned grid = (unsigned)((p.rows + block / p.tpr - 1) / (block / p.tpr));
#define FLAB_NORM(VV, NN) rms_norm_fwd_kernel<T, S, VV, NN, QUANT, NORM><<<grid, block, 0, st>>>(p)
  if (vec) {
    switch (nv) {
      case 1: FLAB_NORM(V, 1); break;
      case 2: FLAB_NORM(V, 2); break;
      case 4: FLAB_NORM(V, 4); break;
      case 8: FLAB_NORM(V, 8); break;
      default: FLAB_NORM(V, 0); break;
    }
  } else if (nv) {
    FLAB_NORM(1, 8);
  } else {
    FLAB_NORM(1, 0);
  }
#undef FLAB_NORM
  return check_launch("rms_norm_fwd");
}

template <typename T, bool QUANT, bool NORM> int norm_fwd_sum(const NormParams &p, bool wide, cudaStream_t st) {
  return wide ? launch_norm_fwd<T, float, QUANT, NORM>(p, st) : launch_norm_fwd<T, T, QUANT, NORM>(p, st);
}

template <typename T> int norm_fwd_typed(const NormParams &p, bool wide, bool quant, bool norm, cudaStream_t st) {
  if (!norm) return launch_norm_fwd<T, T, true, false>(p, st);
  return quant ? norm_fwd_sum<T, true, true>(p, wide, st) : norm_fwd_sum<T, false, true>(p, wide, st);
}

// the shape of a backward launch: everything that its number of partial rows depends on
struct NormBwdPlan {
  int tpr, nv, block, grid;
  bool vec;
};
NormBwdPlan norm_bwd_plan(long long rows, int n, int esize, bool vec) {
  NormBwdPlan q;
  const int V = 16 / esize;
  q.vec = vec && n % V == 0;
  norm_split(rows, q.vec ? n / V : n, q.vec ? 4 : 16, q.tpr, q.nv);
  if (q.tpr > 256) q.tpr = 1024, q.nv = 0;
  q.block = q.nv ? 256 : 1024;
  const long long want = (rows + q.block / q.tpr - 1) / (q.block / q.tpr), cap = (long long)sm_count() * (q.nv ? 3 : 1);
  q.grid = (int)(want < 1 ? 1 : want < cap ? want : cap);
  return q;
}

template <typename T, typename S> int launch_norm_bwd(NormBwdParams p, cudaStream_t st, int &parts) {
  constexpr int V = 16 / sizeof(T);
  const NormBwdPlan q = norm_bwd_plan(p.rows, p.n, sizeof(T), aligned16({p.s, p.dy, p.ds, p.w, p.dx, p.dr}));
  p.tpr = q.tpr;
  parts = q.grid;
  const size_t bytes = p.part ? (size_t)(q.block / q.tpr) * p.n * sizeof(float) : 0;
  FLAB_REQUIRE(bytes <= 227 * 1024 - 1024, FLAB_E_UNSUPPORTED, "rms_norm_bwd: rows of %d elements are not supported", p.n);
#define FLAB_NORM(VV, NN)                                                                                                                   \
  do {                                                                                                                                      \
    auto kernel = rms_norm_bwd_kernel<T, S, VV, NN>;                                                                                        \
    if (bytes > 48 * 1024)                                                                                                                  \
      FLAB_REQUIRE(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess, FLAB_E_LAUNCH,     \
                   "rms_norm_bwd: %zu bytes of shared memory were refused", bytes);                                                         \
    kernel<<<q.grid, q.block, bytes, st>>>(p);                                                                                              \
  } while (0)
  if (q.vec) {
    switch (q.nv) {
      case 1: FLAB_NORM(V, 1); break;
      case 2: FLAB_NORM(V, 2); break;
      case 4: FLAB_NORM(V, 4); break;
      default: FLAB_NORM(V, 0); break;
    }
  } else if (q.nv == 16) {
    FLAB_NORM(1, 16);
  } else if (q.nv) {
    FLAB_NORM(1, 8);
  } else {
    FLAB_NORM(1, 0);
  }
#undef FLAB_NORM
  return check_launch("rms_norm_bwd");
}

}  // namespace

int sum_partials(const float *part, void *out, int parts, int n, int dtype, cudaStream_t st) {
  const int grid = (n + 31) / 32;
  switch (dtype) {
    case FLAB_BF16: partial_sum_kernel<bf16><<<grid, 256, 0, st>>>(part, reinterpret_cast<bf16 *>(out), parts, n); break;
    case FLAB_FP16: partial_sum_kernel<__half><<<grid, 256, 0, st>>>(part, reinterpret_cast<__half *>(out), parts, n); break;
    default: partial_sum_kernel<float><<<grid, 256, 0, st>>>(part, reinterpret_cast<float *>(out), parts, n); break;
  }
  return check_launch("partial_sum");
}

}  // namespace flab

extern "C" {

int flab_rms_norm_fwd(const void *x, const void *residual, const void *weight, void *y, void *sum, float *rstd, float *scale, long long rows, int n,
                      int dtype, int residual_dtype, int sum_dtype, int weight_dtype, int flags, float eps, void *stream) {
  using namespace flab;
  if (rows == 0) return FLAB_OK;
  const bool quant = flags & FLAB_NORM_E4M3, norm = !(flags & FLAB_NORM_NONE);
  FLAB_REQUIRE(x && y && rows > 0 && n > 0, FLAB_E_BADARG, "rms_norm_fwd needs x, y, rows >= 0 and n > 0");
  FLAB_REQUIRE(dtype >= 0 && dtype <= 2 && (sum_dtype == dtype || sum_dtype == FLAB_FP32) && weight_dtype >= 0 && weight_dtype <= 2, FLAB_E_BADARG,
               "rms_norm_fwd: unknown element types %d, %d, %d", dtype, sum_dtype, weight_dtype);
  FLAB_REQUIRE(!residual || residual_dtype == dtype || (residual_dtype == FLAB_FP32 && sum_dtype == FLAB_FP32), FLAB_E_UNSUPPORTED,
               "rms_norm_fwd: a residual of type %d with a sum of type %d is not supported", residual_dtype, sum_dtype);
  FLAB_REQUIRE(norm || (quant && !residual && !weight && !sum && sum_dtype == dtype), FLAB_E_BADARG, "quantisation alone takes x only");
  FLAB_REQUIRE(!quant || scale, FLAB_E_BADARG, "an e4m3 output needs scale");
  FLAB_REQUIRE(rows < (1ll << 31) - 1, FLAB_E_UNSUPPORTED, "rms_norm_fwd: too many rows (%lld)", rows);
  NormParams p = {x, residual, weight, y, sum, rstd, scale, rows, n, 0, residual && residual_dtype == FLAB_FP32 && dtype != FLAB_FP32, weight_dtype, eps};
  const bool wide = sum_dtype == FLAB_FP32;
  switch (dtype) {
    case FLAB_BF16: return norm_fwd_typed<bf16>(p, wide, quant, norm, (cudaStream_t)stream);
    case FLAB_FP16: return norm_fwd_typed<__half>(p, wide, quant, norm, (cudaStream_t)stream);
    default: return norm_fwd_typed<float>(p, false, quant, norm, (cudaStream_t)stream);
  }
}

int flab_rms_norm_partials(long long rows, int n, int dtype) {
  if (rows <= 0 || n <= 0) return 1;
  const int e = dtype == FLAB_FP32 ? 4 : 2;
  const int a = flab::norm_bwd_plan(rows, n, e, true).grid, b = flab::norm_bwd_plan(rows, n, e, false).grid;
  return a > b ? a : b;
}

int flab_rms_norm_bwd(const void *sum, const void *dy, const void *dsum, const void *weight, const float *rstd, void *dx, void *dresidual, void *dweight,
                      float *dw_partial, long long rows, int n, int dtype, int sum_dtype, int weight_dtype, void *stream) {
  using namespace flab;
  cudaStream_t st = (cudaStream_t)stream;
  FLAB_REQUIRE(rows >= 0 && n > 0 && dtype >= 0 && dtype <= 2 && (sum_dtype == dtype || sum_dtype == FLAB_FP32) && weight_dtype >= 0 && weight_dtype <= 2,
               FLAB_E_BADARG, "rms_norm_bwd: unknown element types %d, %d, %d or sizes", dtype, sum_dtype, weight_dtype);
  FLAB_REQUIRE(!dweight || dw_partial, FLAB_E_BADARG, "rms_norm_bwd: dweight needs dw_partial");
  int parts = 0;
  if (rows > 0) {
    FLAB_REQUIRE(sum && dy && rstd && (dx || dresidual || dweight), FLAB_E_BADARG, "rms_norm_bwd needs sum, dy, rstd and an output");
    NormBwdParams p = {sum, dy, dsum, weight, rstd, dx, dresidual, dweight ? dw_partial : nullptr, rows, n, 0, weight_dtype};
    const bool wide = sum_dtype == FLAB_FP32;
    int rc;
    switch (dtype) {
      case FLAB_BF16: rc = wide ? launch_norm_bwd<bf16, float>(p, st, parts) : launch_norm_bwd<bf16, bf16>(p, st, parts); break;
      case FLAB_FP16: rc = wide ? launch_norm_bwd<__half, float>(p, st, parts) : launch_norm_bwd<__half, __half>(p, st, parts); break;
      default: rc = launch_norm_bwd<float, float>(p, st, parts); break;
    }
    if (rc) return rc;
  }
  return dweight ? sum_partials(dw_partial, dweight, parts, n, weight_dtype, st) : FLAB_OK;
}
}
