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
// Measured at 32768 x 2048 bf16 with a residual, of the copy rate: forward 90 us (91 %) in a training step, e4m3 83
// us (87 %), quantised as they are 40 us (77 %), backward 109 us with its partial sums (the kernel alone 102, 80 %); with an fp32 stream
// forward 141 us (87 %), backward 170 (96 %); 256 rows 2.5 us, e4m3 2.9 us, backward 7.4 us (the latency of a row).
// What cannot use the ring is further from its bytes (calls with an empty L2): 2047 x 1111 fp32 16 us forward, 63 backward
// (floor 5.6 each), 8192 x 16384 bf16 223 and 965 us (164 each).  Outside the ring, eight vectors a thread spill 92 to 118 bytes in forward,
// four 72 to 232 in backward.
#include <cuda_fp8.h>

#include <initializer_list>
#include <type_traits>

#include "tc.cuh"

FLAB_TC_DEFINE_ERROR_WORD(rms_norm_error)

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

// Sum over the TPR threads of a row, or the largest |y|: magnitudes go as their bits, whose order is theirs and puts a NaN on top.
// `slot` is a row of shared memory for this reduction, one value a warp of the block; sync() is the barrier of the row's threads.
// Every thread adds the warps' values in the same order.
__device__ __forceinline__ unsigned magnitude(float y) { return __float_as_uint(y) & 0x7fffffffu; }
template <typename Sync> __device__ __forceinline__ float row_sum(float v, int tpr, float *slot, Sync sync) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr > 32) {
    const int nw = tpr >> 5, first = threadIdx.x / tpr * nw, lane = threadIdx.x & 31;
    if (lane == 0) slot[threadIdx.x >> 5] = v;
    sync();
    v = lane < nw ? slot[first + lane] : 0.f;
    for (int o = nw >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    v = __shfl_sync(0xffffffffu, v, 0);
  }
  return v;
}
template <typename Sync> __device__ __forceinline__ float row_top(unsigned v, int tpr, float *slot, Sync sync) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (tpr > 32) {
    const int nw = tpr >> 5, first = threadIdx.x / tpr * nw, lane = threadIdx.x & 31;
    if (lane == 0) slot[threadIdx.x >> 5] = __uint_as_float(v);
    sync();
    v = __reduce_max_sync(0xffffffffu, lane < nw ? __float_as_uint(slot[first + lane]) : 0u);
  }
  return __uint_as_float(v);
}
struct BlockSync {
  __device__ __forceinline__ void operator()() const { __syncthreads(); }
};

// How a row's values become e4m3: divided by the scale where x has 32 bits, so that a value next to the border of two bytes falls as the
// formula has it; multiplied by the scale's reciprocal where x has 16 (an ulp of fp32 is 2^-16 of its step, and the division would
// make the kernel wait for its arithmetic: 87 us with the product against 72 for the bytes at 32768 x 2048).
// A row of zeros has scale 0 and zeros.  Below the normal numbers of fp32 a scale is rounded up where rows are divided by it, so that no
// value passes 448 of them; where they are multiplied it is held at the smallest that has a reciprocal, 2^-126, whose e4m3 steps are below
// those of 16-bit values.  A NaN makes NaNs of its row.  (The rule costs an instruction-bound row something: quantised as they are,
// 131072 x 512 bf16 41.3 -> 43.3 us and 131072 x 256 fp32 33.4 -> 35.2; 32768 x 2048 as before.)
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
template <typename T> struct Quantiser {
  static constexpr bool DIVIDE = sizeof(T) == 4;
  static constexpr float LEAST = 1.17549435e-38f;  // 2^-126
  float by;
  static __device__ __forceinline__ float scale(float top) {
    const float s = top * (1.f / E4M3_MAX);
    return DIVIDE ? (s < LEAST ? __fmul_ru(top, 1.f / E4M3_MAX) : s) : top == 0.f ? 0.f : max_nan(s, LEAST);
  }
  __device__ __forceinline__ Quantiser(float top) : by(DIVIDE ? (top == 0.f ? 1.f : scale(top)) : E4M3_MAX / max_nan(top, E4M3_MAX * LEAST)) {}
  __device__ __forceinline__ float operator()(float y) const { return DIVIDE ? __fdiv_rn(y, by) : y * by; }
};
// V e4m3 bytes, values beyond the type's range held at its largest (a NaN stays one)
template <int V, typename T> __device__ __forceinline__ void store_e4m3(void *base, size_t at, const float (&f)[V], const Quantiser<T> &to) {
  Vec<unsigned char, V> q;
  if constexpr (V == 1) {
    q.v[0] = __nv_cvt_float_to_fp8(to(f[0]), __NV_SATFINITE, __NV_E4M3);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(to(f[j]), to(f[j + 1])), __NV_SATFINITE, __NV_E4M3);
      q.v[j] = two & 0xff, q.v[j + 1] = two >> 8;
    }
  }
  *reinterpret_cast<Vec<unsigned char, V> *>(reinterpret_cast<unsigned char *>(base) + at) = q;
}

// The largest magnitude of 16-bit values, as fp32 bits, two to an instruction: magnitudes go as their bits here as well.
template <typename T, int V> __device__ __forceinline__ unsigned top_of(unsigned most, const Vec<T, V> &v) {
  if constexpr (V == 1) {
    return max(most, (unsigned)(*reinterpret_cast<const unsigned short *>(&v) & 0x7fff));
  } else {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) most = __vmaxu2(most, reinterpret_cast<const unsigned *>(&v)[j] & 0x7fff7fffu);
    return most;
  }
}
template <typename T> __device__ __forceinline__ unsigned wide_top(unsigned most) {
  const unsigned short one = (unsigned short)max(most & 0xffffu, most >> 16);
  return magnitude(Num<T>::f(*reinterpret_cast<const T *>(&one)));
}

// T: x and y;  S: the stored sum;  RES: residual, 0 none, 1 of type T, 2 fp32;  V elements a vector, NV vectors a thread (0: read
// again);  QUANT: e4m3 output;  NORM: without it the rows are quantised as they are.
// All of a row's loads are issued before its first store: with loads and stores of one loop in turn a row was eight trips to
// memory one after the other (2.9 TB/s at 32768 x 2048 bf16).
template <typename T, typename S, int RES, int V, int NV, bool QUANT, bool NORM>
__global__ void __launch_bounds__(NV ? 512 : 1024) rms_norm_fwd_kernel(const NormParams p) {
  typedef typename std::conditional<RES == 2, float, T>::type R;
  __shared__ float slots[2][32];
  const int li = threadIdx.x % p.tpr;
  const long long row = (long long)blockIdx.x * (blockDim.x / p.tpr) + threadIdx.x / p.tpr;
  const bool on = row < p.rows;
  const size_t base = (size_t)row * p.n;
  constexpr int KEEP = NV ? NV : 1;
  const int loops = NV ? NV : (p.n + V * p.tpr - 1) / (V * p.tpr);
  Vec<S, V> s[KEEP];
  auto at = [&](int k) { return (k * p.tpr + li) * V; };
  auto add = [&](const Vec<T, V> &x, const Vec<R, V> &r) {  // the stored sum
    Vec<S, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.v[j] = Num<S>::t(RES ? Num<T>::f(x.v[j]) + Num<R>::f(r.v[j]) : Num<T>::f(x.v[j]));
    return v;
  };
  auto fetch = [&](int c) {
    Vec<T, V> x = *reinterpret_cast<const Vec<T, V> *>(reinterpret_cast<const T *>(p.x) + base + c);
    Vec<R, V> r;
    if (RES) r = *reinterpret_cast<const Vec<R, V> *>(reinterpret_cast<const R *>(p.res) + base + c);
    return add(x, r);
  };
  auto keep_sum = [&](int c, const Vec<S, V> &v) { *reinterpret_cast<Vec<S, V> *>(reinterpret_cast<S *>(p.sum) + base + c) = v; };

  float ss = 0.f;
  if (NV) {
    Vec<T, V> x[KEEP];
    Vec<R, V> r[KEEP];
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      if (on && at(k) < p.n) {
        x[k] = *reinterpret_cast<const Vec<T, V> *>(reinterpret_cast<const T *>(p.x) + base + at(k));
        if (RES) r[k] = *reinterpret_cast<const Vec<R, V> *>(reinterpret_cast<const R *>(p.res) + base + at(k));
      }
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      if (on && at(k) < p.n) {
        s[k] = add(x[k], r[k]);
        if (p.sum) keep_sum(at(k), s[k]);
        if (NORM) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float f = Num<S>::f(s[k].v[j]);
            ss = fmaf(f, f, ss);
          }
        }
      }
  } else if (on && NORM) {
    for (int k = 0; k < loops; ++k)
      if (at(k) < p.n) {
        const Vec<S, V> v = fetch(at(k));
        if (p.sum) keep_sum(at(k), v);
#pragma unroll
        for (int j = 0; j < V; ++j) ss = fmaf(Num<S>::f(v.v[j]), Num<S>::f(v.v[j]), ss);
      }
  }
  float rstd = 1.f;
  if (NORM) {
    ss = row_sum(ss, p.tpr, slots[0], BlockSync());
    rstd = rsqrtf(ss * (1.f / p.n) + p.eps);
    if (on && li == 0 && p.rstd) p.rstd[row] = rstd;
  }
  auto result = [&](int k, float (&y)[V]) {
    const Vec<S, V> v = NV ? s[NV ? k : 0] : fetch(at(k));
    if (!NORM) {
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = Num<S>::f(v.v[j]);
      return;
    }
    float w[V];
    load_w<V>(p.w, p.w_type, at(k), w);
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = Num<S>::f(v.v[j]) * rstd * w[j];
  };
  float top = 0.f;
  if (QUANT) {
    unsigned bits = 0;
#pragma unroll
    for (int k = 0; k < (NV ? NV : loops); ++k)
      if (on && at(k) < p.n) {
        if constexpr (!NORM && sizeof(S) == 2) {
          bits = top_of<S, V>(bits, NV ? s[NV ? k : 0] : fetch(at(k)));
        } else {
          float y[V];
          result(k, y);
#pragma unroll
          for (int j = 0; j < V; ++j) bits = max(bits, magnitude(y[j]));
        }
      }
    if constexpr (!NORM && sizeof(S) == 2) bits = wide_top<S>(bits);
    top = row_top(bits, p.tpr, slots[1], BlockSync());
    if (on && li == 0) p.scale[row] = Quantiser<T>::scale(top);
  }
  const Quantiser<T> to(top);
#pragma unroll
  for (int k = 0; k < (NV ? NV : loops); ++k)
    if (on && at(k) < p.n) {
      float y[V];
      result(k, y);
      if constexpr (QUANT) store_e4m3<V>(p.y, base + at(k), y, to);
      else store_f<T, V>(p.y, base + at(k), y);
    }
}

struct NormBwdParams {
  const void *s, *dy, *ds, *w;
  const float *rstd;
  void *dx, *dr;
  float *part;
  long long rows;
  int n, tpr, w_type;
  int in_place;  // rows too long for shared memory: dw is summed in the partial row itself
};

// one partial row of dw a block; the block's groups of TPR threads take rows in turn
template <typename T, typename S, int V, int NV> __global__ void __launch_bounds__(NV ? 256 : 1024, NV ? 2 : 1) rms_norm_bwd_kernel(const NormBwdParams p) {
  extern __shared__ float sdw[];  // [groups][n]
  __shared__ float slots[2][32];
  const int li = threadIdx.x % p.tpr, group = threadIdx.x / p.tpr, groups = blockDim.x / p.tpr;
  constexpr int KEEP = NV ? NV : 1;
  const int loops = NV ? NV : (p.n + V * p.tpr - 1) / (V * p.tpr);
  float acc[KEEP][V] = {};
  // rows too long for registers: the thread's columns are its own in shared memory, or in its block's partial row (one group a block)
  float *const own = p.part + (size_t)blockIdx.x * p.n;
  if (!NV && p.part) {
    for (int k = 0; k < loops; ++k)
      for (int j = 0; j < V; ++j) {
        const int c = (k * p.tpr + li) * V + j;
        if (c >= p.n) continue;
        if (p.in_place) own[c] = 0.f;
        else sdw[c] = 0.f;
      }
  }
  int par = 0;
  for (long long r0 = (long long)blockIdx.x * groups; r0 < p.rows; r0 += (long long)gridDim.x * groups, par ^= 1) {
    const long long row = r0 + group;
    const bool on = row < p.rows;
    const size_t base = (size_t)row * p.n;
    const float rstd = on ? p.rstd[row] : 0.f;
    Vec<S, V> s[KEEP], ds[KEEP];
    Vec<T, V> dy[KEEP];
    float dot = 0.f;
    auto at = [&](int k) { return (k * p.tpr + li) * V; };
    auto fetch = [&](int i, int c) {
      s[i] = *reinterpret_cast<const Vec<S, V> *>(reinterpret_cast<const S *>(p.s) + base + c);
      dy[i] = *reinterpret_cast<const Vec<T, V> *>(reinterpret_cast<const T *>(p.dy) + base + c);
      if (p.ds) ds[i] = *reinterpret_cast<const Vec<S, V> *>(reinterpret_cast<const S *>(p.ds) + base + c);
    };
    if (NV) {  // all of a row's loads first
#pragma unroll
      for (int k = 0; k < KEEP; ++k)
        if (on && at(k) < p.n) fetch(k, at(k));
    }
#pragma unroll
    for (int k = 0; k < (NV ? NV : loops); ++k)
      if (on && at(k) < p.n) {
        const int c = at(k), i = NV ? k : 0;
        if (!NV) fetch(0, c);
        float w[V];
        load_w<V>(p.w, p.w_type, c, w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = Num<S>::f(s[i].v[j]) * rstd, d = Num<T>::f(dy[i].v[j]);
          dot = fmaf(xh, w[j] * d, dot);
          if (NV) acc[i][j] = fmaf(d, xh, acc[i][j]);
          else if (p.in_place) own[c + j] = fmaf(d, xh, own[c + j]);
          else if (p.part) sdw[c + j] = fmaf(d, xh, sdw[c + j]);
        }
      }
    dot = row_sum(dot, p.tpr, slots[par], BlockSync()) / p.n;
#pragma unroll
    for (int k = 0; k < (NV ? NV : loops); ++k)
      if (on && at(k) < p.n) {
        const int c = at(k), i = NV ? k : 0;
        if (!NV) fetch(0, c);
        float w[V], d[V];
        load_w<V>(p.w, p.w_type, c, w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          d[j] = (w[j] * Num<T>::f(dy[i].v[j]) - Num<S>::f(s[i].v[j]) * rstd * dot) * rstd;
          if (p.ds) d[j] += Num<S>::f(ds[i].v[j]);
        }
        if (p.dx) store_f<T, V>(p.dx, base + c, d);
        if (p.dr) store_f<S, V>(p.dr, base + c, d);
      }
  }
  if (!p.part || (!NV && p.in_place)) return;
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

// ---- many rows: a persistent block, rows by bulk copies -----------------------------------------------------------------
// A group of TPR threads walks rows through a ring of shared-memory stages that its first thread keeps filled, so that loads
// stay in flight over the reductions and stores of the rows before; a thread holds its columns' weights (and, in backward, their
// dw) in registers for all its rows.  The reduction of a row is also the point behind which its stage may be refilled: forward's takes in
// all that was read of the stage.  Backward's does not take in the stream's gradient, and a row of one warp reduces by shuffles alone,
// so a barrier of the warp stands there as well.
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(tc::smem_u32(bar))
               : "memory");
}

constexpr int RING_THREADS = 512, MAX_STAGES = 8;

struct RingShape {
  int tpr, groups, stages, row_bytes;
};

// the barrier of a group's threads
struct GroupSync {
  int tpr, group;
  __device__ __forceinline__ void operator()() const {
    if (tpr == RING_THREADS) __syncthreads();
    else tc::named_barrier(1 + group, tpr);
  }
};

template <typename T, typename S, int RES, int NV, bool QUANT>
__global__ void __launch_bounds__(RING_THREADS, 1) rms_norm_fwd_ring_kernel(const NormParams p, const RingShape q) {
  typedef typename std::conditional<RES == 2, float, T>::type R;
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(128) char ring[];
  __shared__ uint64_t full[16][MAX_STAGES];
  __shared__ float slots[4][RING_THREADS / 32];
  const int group = threadIdx.x / q.tpr, li = threadIdx.x % q.tpr;
  char *const mine = ring + (size_t)group * q.stages * q.row_bytes;
  if (li == 0)
    for (int i = 0; i < q.stages; ++i) tc::mbar_init(&full[group][i], 1);
  tc::fence_barrier_init();
  __syncthreads();
  const long long row0 = (long long)blockIdx.x * q.groups + group, stride = (long long)gridDim.x * q.groups;
  const uint32_t x_bytes = p.n * sizeof(T), r_bytes = RES ? p.n * sizeof(R) : 0;
  auto fill = [&](int st, long long row) {
    char *dst = mine + (size_t)st * q.row_bytes;
    tc::mbar_expect_tx(&full[group][st], x_bytes + r_bytes);
    bulk_load(dst, reinterpret_cast<const T *>(p.x) + row * p.n, x_bytes, &full[group][st]);
    if (RES) bulk_load(dst + x_bytes, reinterpret_cast<const R *>(p.res) + row * p.n, r_bytes, &full[group][st]);
  };
  if (li == 0)
    for (int i = 0; i < q.stages; ++i)
      if (row0 + i * stride < p.rows) fill(i, row0 + i * stride);
  auto at = [&](int k) { return (k * q.tpr + li) * V; };
  float w[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (at(k) < p.n) load_w<V>(p.w, p.w_type, at(k), w[k]);
  bool dead = false;
  int st = 0, phase = 0, par = 0;
  for (long long row = row0; row < p.rows; row += stride, par ^= 1) {
    const char *src = mine + (size_t)st * q.row_bytes;
    if (!dead && !tc::mbar_wait(&full[group][st], phase)) tu_tc_error = 720, dead = true;
    const size_t base = (size_t)row * p.n;
    Vec<S, V> s[NV];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (at(k) < p.n) {
        const Vec<T, V> x = *reinterpret_cast<const Vec<T, V> *>(src + at(k) * sizeof(T));
        Vec<R, V> r;
        if (RES) r = *reinterpret_cast<const Vec<R, V> *>(src + x_bytes + at(k) * sizeof(R));
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s[k].v[j] = Num<S>::t(RES ? Num<T>::f(x.v[j]) + Num<R>::f(r.v[j]) : Num<T>::f(x.v[j]));
          const float f = Num<S>::f(s[k].v[j]);
          ss = fmaf(f, f, ss);
        }
      }
    ss = row_sum(ss, q.tpr, slots[par], GroupSync{q.tpr, group});
    if (li == 0 && !dead && row + q.stages * stride < p.rows) fill(st, row + q.stages * stride);
    if (++st == q.stages) st = 0, phase ^= 1;
    const float rstd = rsqrtf(ss * (1.f / p.n) + p.eps);
    if (li == 0 && p.rstd) p.rstd[row] = rstd;
    if (p.sum) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (at(k) < p.n) *reinterpret_cast<Vec<S, V> *>(reinterpret_cast<S *>(p.sum) + base + at(k)) = s[k];
    }
    // The products that an e4m3 row needs twice are kept where the sum has 16 bits (32768 x 2048 bf16, cold: 91 -> 87 us) and formed again
    // where it has 32 (with an fp32 residual 123 us, and 131 kept).
    constexpr bool ONCE = QUANT && sizeof(S) == 2;
    float top = 0.f, kept[ONCE ? NV : 1][V];
    auto result = [&](int k, int j) { return Num<S>::f(s[k].v[j]) * rstd * w[k][j]; };
    if (ONCE) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) kept[ONCE ? k : 0][j] = result(k, j);
    }
    if (QUANT) {
      unsigned bits = 0;
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (at(k) < p.n) {
#pragma unroll
          for (int j = 0; j < V; ++j) bits = max(bits, magnitude(ONCE ? kept[ONCE ? k : 0][j] : result(k, j)));
        }
      top = row_top(bits, q.tpr, slots[2 + par], GroupSync{q.tpr, group});
      if (li == 0) p.scale[row] = Quantiser<T>::scale(top);
    }
    const Quantiser<T> to(top);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (at(k) < p.n) {
        float y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = ONCE ? kept[ONCE ? k : 0][j] : result(k, j);
        if constexpr (QUANT) store_e4m3<V>(p.y, base + at(k), y, to);
        else store_f<T, V>(p.y, base + at(k), y);
      }
  }
}

template <typename T, typename S, int NV> __global__ void __launch_bounds__(RING_THREADS, 1) rms_norm_bwd_ring_kernel(const NormBwdParams p, const RingShape q) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(128) char ring[];
  __shared__ uint64_t full[16][MAX_STAGES];
  __shared__ float slots[2][RING_THREADS / 32];
  const int group = threadIdx.x / q.tpr, li = threadIdx.x % q.tpr;
  char *const mine = ring + (size_t)group * q.stages * q.row_bytes;
  if (li == 0)
    for (int i = 0; i < q.stages; ++i) tc::mbar_init(&full[group][i], 1);
  tc::fence_barrier_init();
  __syncthreads();
  const long long row0 = (long long)blockIdx.x * q.groups + group, stride = (long long)gridDim.x * q.groups;
  const uint32_t s_bytes = p.n * sizeof(S), y_bytes = p.n * sizeof(T);
  auto fill = [&](int st, long long row) {
    char *dst = mine + (size_t)st * q.row_bytes;
    tc::mbar_expect_tx(&full[group][st], y_bytes + (p.ds ? 2 : 1) * s_bytes);
    bulk_load(dst, reinterpret_cast<const S *>(p.s) + row * p.n, s_bytes, &full[group][st]);
    bulk_load(dst + s_bytes, reinterpret_cast<const T *>(p.dy) + row * p.n, y_bytes, &full[group][st]);
    if (p.ds) bulk_load(dst + s_bytes + y_bytes, reinterpret_cast<const S *>(p.ds) + row * p.n, s_bytes, &full[group][st]);
  };
  if (li == 0)
    for (int i = 0; i < q.stages; ++i)
      if (row0 + i * stride < p.rows) fill(i, row0 + i * stride);
  auto at = [&](int k) { return (k * q.tpr + li) * V; };
  float w[NV][V], acc[NV][V] = {};
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (at(k) < p.n) load_w<V>(p.w, p.w_type, at(k), w[k]);
  bool dead = false;
  int st = 0, phase = 0, par = 0;
  for (long long row = row0; row < p.rows; row += stride, par ^= 1) {
    const char *src = mine + (size_t)st * q.row_bytes;
    const float rstd = p.rstd[row];
    if (!dead && !tc::mbar_wait(&full[group][st], phase)) tu_tc_error = 721, dead = true;
    const size_t base = (size_t)row * p.n;
    Vec<S, V> s[NV], ds[NV];
    Vec<T, V> dy[NV];
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (at(k) < p.n) {
        s[k] = *reinterpret_cast<const Vec<S, V> *>(src + at(k) * sizeof(S));
        dy[k] = *reinterpret_cast<const Vec<T, V> *>(src + s_bytes + at(k) * sizeof(T));
        if (p.ds) ds[k] = *reinterpret_cast<const Vec<S, V> *>(src + s_bytes + y_bytes + at(k) * sizeof(S));
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = Num<S>::f(s[k].v[j]) * rstd, d = Num<T>::f(dy[k].v[j]);
          dot = fmaf(xh, w[k][j] * d, dot);
          acc[k][j] = fmaf(d, xh, acc[k][j]);
        }
      }
    dot = row_sum(dot, q.tpr, slots[par], GroupSync{q.tpr, group}) / p.n;
    __syncwarp();  // (all lanes have read ds)
    if (li == 0 && !dead && row + q.stages * stride < p.rows) fill(st, row + q.stages * stride);
    if (++st == q.stages) st = 0, phase ^= 1;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (at(k) < p.n) {
        float d[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          d[j] = (w[k][j] * Num<T>::f(dy[k].v[j]) - Num<S>::f(s[k].v[j]) * rstd * dot) * rstd;
          if (p.ds) d[j] += Num<S>::f(ds[k].v[j]);
        }
        if (p.dx) store_f<T, V>(p.dx, base + at(k), d);
        if (p.dr) store_f<S, V>(p.dr, base + at(k), d);
      }
  }
  if (!p.part) return;
  __syncthreads();  // the ring is empty: every row that was asked for has been read
  float *const sdw = reinterpret_cast<float *>(ring);
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (at(k) < p.n) {
#pragma unroll
      for (int j = 0; j < V; ++j) sdw[(size_t)group * p.n + at(k) + j] = acc[k][j];
    }
  __syncthreads();
  for (int c = threadIdx.x; c < p.n; c += RING_THREADS) {
    float t = 0.f;
    for (int i = 0; i < q.groups; ++i) t += sdw[(size_t)i * p.n + c];
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

bool aligned_to(int bytes, std::initializer_list<const void *> ptrs) {
  for (const void *q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % bytes != 0) return false;
  return true;
}
bool aligned16(std::initializer_list<const void *> ptrs) { return aligned_to(16, ptrs); }

// The ring's shape for rows of n elements (V a vector) of which a stage holds row_bytes; false: not for these rows.  `per` is how many
// vectors a thread is to have, `most` how many it can.  Few are quick over a row, many let more groups have rows in hand, which is what
// counts where a row has a second reduction (e4m3) or a longer way (backward).  Us with 8 / 16 / 32 elements a thread: e4m3 32768 x 2048
// bf16 121 / 87 / 83, 16384 x 8192 bf16 - / 177 / 150, with an fp32 residual 141 / 124 / 144; backward 32768 x 2048 bf16 140 / 109 /
// 224 (spilled), 16384 x 2048 fp32 128, 89 and 71 with 4, 8 and 16.
// The ring pays from so many rows a group on (`enough`, at two vectors a thread): forward at 2048 columns of bf16, 2368 rows 9.0 us
// against 8.8 without it, 4096 rows 13.4 against 15.0, 32768 rows 78 against 98; backward 1184 rows 10.5 against 15.1, 32768 rows 102
// against 213.
bool ring_shape(long long rows, int n, int V, long long row_bytes, int enough, int per, int most, RingShape &q, int &nv, int &grid) {
  constexpr int RING = 200 * 1024;
  if (2 * row_bytes > RING) return false;
  const int vecs = n / V;
  q.tpr = 32;
  while (per * q.tpr < vecs && q.tpr < RING_THREADS) q.tpr *= 2;
  nv = (vecs + q.tpr - 1) / q.tpr;
  if (nv == 3) nv = 4;
  q.groups = RING_THREADS / q.tpr;
  q.row_bytes = (int)row_bytes;
  q.stages = (int)(RING / (q.groups * row_bytes));
  if (q.stages > MAX_STAGES) q.stages = MAX_STAGES;
  grid = sm_count();
  const int have = per > 2 && nv < per ? 2 : per;
  return nv <= most && q.stages >= 2 && rows * have >= 2ll * enough * q.groups * grid;
}

template <typename T, typename S, int RES, bool QUANT, bool NORM> int launch_norm_fwd(NormParams p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  int nv = 0;
  const bool aligned = p.n % V == 0 && aligned16({p.x, p.res, p.w, p.y, p.sum});
  RingShape q;
  int grid_ring;
  const long long row_bytes = p.n * (long long)(sizeof(T) + (RES == 2 ? 4 : RES ? sizeof(T) : 0));
  // Forward has one reduction: 16 elements a thread for 16 bits (32768 x 2048 90 us against 99 with 8, in a training step), and for 32 bits
  // 8 where the inputs may still lie in L2 (below its 126 MB: 2368 x 2048 11.0 us against 13.6) and 4 from HBM (16384 x 2048 98 and 85).
  const int per = QUANT ? (sizeof(S) == 2 ? 32 : 16) / V : sizeof(T) == 4 && p.rows * row_bytes >= 1ll << 27 ? 1 : 2;
  if (NORM && aligned && ring_shape(p.rows, p.n, V, row_bytes, 6, per, QUANT || V == 4 ? 4 : 2, q, nv, grid_ring)) {
    const size_t bytes = (size_t)q.groups * q.stages * q.row_bytes;
    auto launch = [&](auto kernel) {
      const int rc = set_smem(kernel, bytes);
      if (rc) return rc;
      kernel<<<grid_ring, RING_THREADS, bytes, st>>>(p, q);
      return check_launch("rms_norm_fwd");
    };
    if constexpr (QUANT || V == 4) {
      if (nv == 4) return launch(rms_norm_fwd_ring_kernel<T, S, RES, 4, QUANT>);
    }
    return nv == 1 ? launch(rms_norm_fwd_ring_kernel<T, S, RES, 1, QUANT>) : launch(rms_norm_fwd_ring_kernel<T, S, RES, 2, QUANT>);
  }
  nv = 0;
  int by = aligned ? V : p.n % 2 == 0 && aligned_to(8, {p.x, p.res, p.w, p.y, p.sum}) ? 2 : 1;  // elements a load
  norm_split(p.rows, p.n / by, 8, p.tpr, nv);
  if (nv == 0 && by > 1) by = 1, norm_split(p.rows, p.n, 8, p.tpr, nv);
  const int block = p.tpr < 128 ? 128 : p.tpr;
  const unsigned grid = (unsigned)((p.rows + block / p.tpr - 1) / (block / p.tpr));
#define FLAB_NORM(VV, NN) rms_norm_fwd_kernel<T, S, RES, VV, NN, QUANT, NORM><<<grid, block, 0, st>>>(p)
  if (by == V) {
    switch (nv) {
      case 1: FLAB_NORM(V, 1); break;
      case 2: FLAB_NORM(V, 2); break;
      case 4: FLAB_NORM(V, 4); break;
      default: FLAB_NORM(V, 8); break;
    }
  } else if (by == 2) {
    FLAB_NORM(2, 8);
  } else if (nv) {
    FLAB_NORM(1, 8);
  } else {
    FLAB_NORM(1, 0);
  }
#undef FLAB_NORM
  return check_launch("rms_norm_fwd");
}

template <typename T, bool QUANT> int norm_fwd_sum(const NormParams &p, bool wide, cudaStream_t st) {
  if (!wide) return p.res ? launch_norm_fwd<T, T, 1, QUANT, true>(p, st) : launch_norm_fwd<T, T, 0, QUANT, true>(p, st);
  if (!p.res) return launch_norm_fwd<T, float, 0, QUANT, true>(p, st);
  if constexpr (sizeof(T) == 2) {
    if (p.res_fp32) return launch_norm_fwd<T, float, 2, QUANT, true>(p, st);
  }
  return launch_norm_fwd<T, float, 1, QUANT, true>(p, st);
}

template <typename T> int norm_fwd_typed(const NormParams &p, bool wide, bool quant, bool norm, cudaStream_t st) {
  if (!norm) return launch_norm_fwd<T, T, 0, true, false>(p, st);
  return quant ? norm_fwd_sum<T, true>(p, wide, st) : norm_fwd_sum<T, false>(p, wide, st);
}

// the shape of a backward launch: everything that its number of partial rows depends on
struct NormBwdPlan {
  int by, tpr, nv, block, grid;  // elements a load, threads a row, vectors a thread
};
NormBwdPlan norm_bwd_plan(long long rows, int n, int esize, int by) {
  NormBwdPlan q;
  q.by = by;
  norm_split(rows, n / by, by == 16 / esize ? 4 : by == 2 ? 8 : 16, q.tpr, q.nv);
  if (q.nv == 0 || q.tpr > 256) {
    if (by > 1) return norm_bwd_plan(rows, n, esize, 1);
    q.tpr = 1024, q.nv = 0;
  }
  q.block = q.nv ? 256 : 1024;
  const long long want = (rows + q.block / q.tpr - 1) / (q.block / q.tpr), cap = (long long)sm_count() * (q.nv ? 2 : 1);
  q.grid = (int)(want < 1 ? 1 : want < cap ? want : cap);
  return q;
}

template <typename T, typename S> int launch_norm_bwd(NormBwdParams p, cudaStream_t st, int &parts) {
  constexpr int V = 16 / sizeof(T);
  const bool aligned = aligned16({p.s, p.dy, p.ds, p.w, p.dx, p.dr});
  RingShape r;
  int nv;
  if (aligned && p.n % V == 0 && ring_shape(p.rows, p.n, V, p.n * (long long)(sizeof(T) + 2 * sizeof(S)), 2, 16 / V, 16 / V, r, nv, parts)) {
    size_t bytes = (size_t)r.groups * r.stages * r.row_bytes;
    const size_t sums = (size_t)r.groups * p.n * sizeof(float);
    if (bytes < sums) bytes = sums;
    auto launch = [&](auto kernel) {
      const int rc = set_smem(kernel, bytes);
      if (rc) return rc;
      kernel<<<parts, RING_THREADS, bytes, st>>>(p, r);
      return check_launch("rms_norm_bwd");
    };
    if constexpr (V == 4) {
      if (nv == 4) return launch(rms_norm_bwd_ring_kernel<T, S, 4>);
    }
    return nv == 1 ? launch(rms_norm_bwd_ring_kernel<T, S, 1>) : launch(rms_norm_bwd_ring_kernel<T, S, 2>);
  }
  const int by = aligned && p.n % V == 0 ? V : p.n % 2 == 0 && aligned_to(8, {p.s, p.dy, p.ds, p.w, p.dx, p.dr}) ? 2 : 1;
  const NormBwdPlan q = norm_bwd_plan(p.rows, p.n, sizeof(T), by);
  p.tpr = q.tpr;
  parts = q.grid;
  size_t bytes = p.part ? (size_t)(q.block / q.tpr) * p.n * sizeof(float) : 0;
  // (from 57857 elements on, at four bytes a column; what fits registers is far below: 16384 columns)
  if (bytes > 227 * 1024 - 1024) p.in_place = 1, bytes = 0;
#define FLAB_NORM(VV, NN)                                                                                                                   \
  do {                                                                                                                                      \
    auto kernel = rms_norm_bwd_kernel<T, S, VV, NN>;                                                                                        \
    const int rc = set_smem(kernel, bytes);                                                                                                 \
    if (rc) return rc;                                                                                                                      \
    kernel<<<q.grid, q.block, bytes, st>>>(p);                                                                                              \
  } while (0)
  if (q.by == V) {
    switch (q.nv) {
      case 1: FLAB_NORM(V, 1); break;
      case 2: FLAB_NORM(V, 2); break;
      default: FLAB_NORM(V, 4); break;
    }
  } else if (q.by == 2) {
    FLAB_NORM(2, 8);
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
  FLAB_REQUIRE(rows < (1ll << 31) - 1 && n <= 1 << 30, FLAB_E_UNSUPPORTED, "rms_norm_fwd: too many rows (%lld) or columns (%d)", rows, n);
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
  int most = flab::sm_count();  // the ring's grid
  for (int by : {16 / e, 2, 1}) {
    if (n % by) continue;
    const int grid = flab::norm_bwd_plan(rows, n, e, by).grid;
    most = grid > most ? grid : most;
  }
  return most;
}

int flab_rms_norm_bwd(const void *sum, const void *dy, const void *dsum, const void *weight, const float *rstd, void *dx, void *dresidual, void *dweight,
                      float *dw_partial, long long rows, int n, int dtype, int sum_dtype, int weight_dtype, void *stream) {
  using namespace flab;
  cudaStream_t st = (cudaStream_t)stream;
  FLAB_REQUIRE(rows >= 0 && n > 0 && dtype >= 0 && dtype <= 2 && (sum_dtype == dtype || sum_dtype == FLAB_FP32) && weight_dtype >= 0 && weight_dtype <= 2,
               FLAB_E_BADARG, "rms_norm_bwd: unknown element types %d, %d, %d or sizes", dtype, sum_dtype, weight_dtype);
  FLAB_REQUIRE(n <= 1 << 30, FLAB_E_UNSUPPORTED, "rms_norm_bwd: too many columns (%d)", n);
  FLAB_REQUIRE(!dweight || dw_partial, FLAB_E_BADARG, "rms_norm_bwd: dweight needs dw_partial");
  int parts = 0;
  if (rows > 0) {
    FLAB_REQUIRE(sum && dy && rstd && (dx || dresidual || dweight), FLAB_E_BADARG, "rms_norm_bwd needs sum, dy, rstd and an output");
    NormBwdParams p = {sum, dy, dsum, weight, rstd, dx, dresidual, dweight ? dw_partial : nullptr, rows, n, 0, weight_dtype, 0};
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
