// Element-wise gated linear recurrence over time (the HGRN family; fla/ops/hgrn/{chunk,fused_recurrent}.py), forward and
// backward, for fixed-length batches [B, T, D] and for sequences packed into one row with cumulative lengths.
//   forward :  h_t = e^{g_t} h_{t-1} + x_t,  o_t = h_t            (h before a sequence: its h0, or 0;  ht = its last h)
//   backward:  c_t = e^{g_t} (do_t + c_{t+1}),  dx_t = do_t + c_{t+1},  dg_t = c_t h_{t-1},  dh0 = c at the first token
//              (c behind a sequence: the gradient of its ht, or 0)
// c_t is the gradient with respect to h_{t-1}, so both directions are the same affine recurrence y <- P y + Q and compose:
// (P2, Q2) o (P1, Q1) = (P2 P1, P2 Q1 + Q2).  A sequence's edge is the map (0, h0).
//
// Bound by HBM: x, g in and o out, once (g, o, do in and dx, dg out).  A block owns a tile of L tokens x C channels and keeps
// it in registers: each warp composes R consecutive rows (lanes side by side over the channels), the warps' maps are joined
// through shared memory, and the tile's start value comes from the tiles before it: every tile publishes its map, the last tile
// of each group of G publishes the group's end value, and a tile takes the end of the group before its own through the maps of
// its group's earlier tiles.  The sums are formed in the same order whatever block runs when, so results repeat bit for bit (a
// look-back that takes whatever is there first would be no faster and would not).  Serial along time is one hop a group: a word
// of 64 bits that holds value and mark.  Tiles are handed out by a ticket in the order of time, so that a tile waits only for
// tiles whose blocks already run; one launch then reads everything once, where a two-pass scan would read the inputs twice.
// All arithmetic and every state is fp32; o, dx, dg are rounded once, when stored.  Backward takes h_{t-1} from the stored o:
// dg is a plain product with it, so the 16-bit rounding of o enters dg once, with the size of dg's own rounding, and backward
// needs neither x nor a second forward scan.
#include "tc.cuh"

FLAB_TC_DEFINE_ERROR_WORD(hgrn_error)

namespace flab {
namespace {

constexpr int G = 8;  // tiles of a group

enum { ROW_START = 1, ROW_END = 2, ROW_OUT = 4, ROW_SHIFT = 3 };

struct HgrnParams {
  const void *x;     // fwd: x;  bwd: do
  const void *g;
  const void *o_in;  // bwd: forward output
  const float *h0;   // fwd and bwd (h before the sequence), may be null
  const float *dht;  // bwd, may be null
  void *o;           // fwd: o;  bwd: dx
  void *dg;
  float *ht;         // fwd: ht;  bwd: dh0;  may be null
  const void *cu;
  int cu64;
  int B, D, N;
  int nT, nCG;       // tiles along time, channel groups
  long long T;
  int *flags;        // [tiles] 1: the tile's map is there; null with one tile along time
  int *ticket;
  float2 *maps;      // [tiles][C] (P, Q)
  unsigned long long *ends;  // [groups][C] end value and mark
};

template <typename T, int V> struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

__device__ __forceinline__ long long cu_at(const HgrnParams &p, int n) {
  return p.cu64 ? reinterpret_cast<const long long *>(p.cu)[n] : (long long)reinterpret_cast<const int *>(p.cu)[n];
}

// Row t of a packed batch: which sequence's first / last row it is, if any.  The sequence is the last one that begins at or
// before t, so empty sequences at the same place are passed over.
__device__ __forceinline__ int row_code(const HgrnParams &p, long long t) {
  int lo = 0, hi = p.N + 1;  // number of cumulative lengths that are <= t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu_at(p, mid) <= t) lo = mid + 1;
    else hi = mid;
  }
  const int n = lo - 1;
  if (n < 0 || n >= p.N) return ROW_OUT;
  return (n << ROW_SHIFT) | (cu_at(p, n) == t ? ROW_START : 0) | (cu_at(p, n + 1) == t + 1 ? ROW_END : 0);
}

// The factor of a map that holds a sequence's edge: nothing of what comes before gets through it, not even a NaN or an
// infinity.  Gates are exponentials, so no other factor has a sign; one that underflowed to +0 still hands a NaN on.
#define CUT (-0.f)
__device__ __forceinline__ bool is_cut(float P) { return __float_as_uint(P) == 0x80000000u; }
// y = P c + Q.  A zero start stays out of the product, so that a P that overflowed (gates above 0) makes no NaN of it.
__device__ __forceinline__ float through(float P, float Q, float c) { return c == 0.f || is_cut(P) ? Q : fmaf(P, c, Q); }

__device__ __forceinline__ int load_acquire(const int *a) {
  int v;
  asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(a) : "memory");
  return v;
}
__device__ __forceinline__ void store_release(int *a, int v) {
  asm volatile("st.release.gpu.global.b32 [%0], %1;" ::"l"(a), "r"(v) : "memory");
}
// Bounded wait for a tile's flag: about a second; once any wait has run out, no further one waits.
__device__ __forceinline__ int wait_flag(const int *a) {
  int v = load_acquire(a);
  if (v) return v;
  const long long t0 = clock64();
  for (int spins = 1;; ++spins) {
    v = load_acquire(a);
    if (v) return v;
    if ((spins & 255) == 0 && (clock64() - t0 > (1ll << 31) || *reinterpret_cast<volatile int *>(&tu_tc_error))) {
      tu_tc_error = 700;
      return 0;
    }
  }
}

// A group's end value and the mark that it is there, in one word of 64 bits: whoever sees the mark has the value.
__device__ __forceinline__ void put_end(unsigned long long *a, float v) {
  const unsigned long long word = (1ull << 32) | __float_as_uint(v);
  asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(a), "l"(word) : "memory");
}
__device__ __forceinline__ float wait_end(const unsigned long long *a) {
  unsigned long long v;
  const long long t0 = clock64();
  for (int spins = 1;; ++spins) {
    asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(v) : "l"(a) : "memory");
    if (v >> 32) break;
    if ((spins & 255) == 0 && (clock64() - t0 > (1ll << 31) || *reinterpret_cast<volatile int *>(&tu_tc_error))) {
      tu_tc_error = 701;
      break;
    }
  }
  return __uint_as_float((unsigned)v);
}

template <typename T, int V, int W, int R, bool BWD, bool VAR>
__global__ void __launch_bounds__(W * 32, 2) hgrn_tile_kernel(const HgrnParams p) {
  constexpr int C = 32 * V, L = W * R;
  __shared__ float sP[W][C], sQ[W][C];
  __shared__ float lP[G - 1][C], lQ[G - 1][C];
  static_assert(W >= G - 1, "a warp for each earlier tile of a group");
  __shared__ int sCode[VAR ? L : 1];
  __shared__ int sTile;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int tile = blockIdx.x;
  if (p.flags) {
    if (threadIdx.x == 0) sTile = atomicAdd(p.ticket, 1);
    __syncthreads();
    tile = sTile;
  }
  const int chains = p.B * p.nCG, step = tile / chains, chain = tile - step * chains;  // step: position along the scan
  const int b = chain / p.nCG, ch = (chain - b * p.nCG) * C + lane * V;
  const bool on = ch < p.D;
  const long long tile0 = (long long)(BWD ? p.nT - 1 - step : step) * L;  // first token of the tile
  const int rows = p.T - tile0 < L ? (int)(p.T - tile0) : L;
  const size_t base = ((size_t)b * p.T + tile0) * p.D + ch;
  const T *const xp = reinterpret_cast<const T *>(p.x) + base, *const gp = reinterpret_cast<const T *>(p.g) + base;
  const T *const op = reinterpret_cast<const T *>(p.o_in) + base;
  T *const yp = reinterpret_cast<T *>(p.o) + base, *const zp = reinterpret_cast<T *>(p.dg) + base;

  // position s = w R + r of the scan is row s of the tile, counted from the tile's end in backward
  auto row = [&](int r) -> int { return BWD ? L - 1 - (w * R + r) : w * R + r; };
  typedef Pack<T, V> PV;
  PV xv[R], gv[R], ov[BWD ? R : 1];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int t = row(r);
    if (t < rows && on) {
      const int at = t * p.D;  // L D < 2^31
      gv[r] = *reinterpret_cast<const PV *>(gp + at);
      xv[r] = *reinterpret_cast<const PV *>(xp + at);
      if (BWD && (t > 0 || tile0 > 0)) ov[r] = *reinterpret_cast<const PV *>(op + (at - p.D));
    }
  }
  if (VAR) {
    for (int s = threadIdx.x; s < L; s += W * 32) sCode[s] = s < rows ? row_code(p, tile0 + s) : ROW_OUT;
    __syncthreads();
  }
  // the warp's own map
  const float *edge = BWD ? p.dht : p.h0;  // value in front of a sequence, in scan order
  float a[R][V], P[V], Q[V];
#pragma unroll
  for (int j = 0; j < V; ++j) P[j] = 1.f, Q[j] = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int t = row(r);
    bool live = t < rows && on;
    if (VAR) {
      const int code = sCode[t];
      live = live && !(code & ROW_OUT);
      if (code & (ROW_OUT | (BWD ? ROW_END : ROW_START))) {
#pragma unroll
        for (int j = 0; j < V; ++j) P[j] = CUT, Q[j] = (code & ROW_OUT) || !edge || !on ? 0.f : edge[(size_t)(code >> ROW_SHIFT) * p.D + ch + j];
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      a[r][j] = live ? expf(Num<T>::f(gv[r].v[j])) : 1.f;
      const float in = live ? Num<T>::f(xv[r].v[j]) : 0.f;
      Q[j] = BWD ? a[r][j] * (Q[j] + in) : fmaf(a[r][j], Q[j], in);
      P[j] *= a[r][j];
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) sP[w][lane * V + j] = P[j], sQ[w][lane * V + j] = Q[j];
  __syncthreads();

  auto joined = [&](int j) -> float2 {  // the tile's map of channel j of this lane
    float jP = 1.f, jQ = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float Pi = sP[i][lane * V + j];
      jQ = through(Pi, sQ[i][lane * V + j], jQ);
      jP = is_cut(Pi) ? CUT : jP * Pi;
    }
    return make_float2(jP, jQ);
  };

  // the tile's start value: the end of the group of tiles before its own, taken through the maps of its group's earlier tiles
  float c[V];
#pragma unroll
  for (int j = 0; j < V; ++j) c[j] = !VAR && step < G && edge && on ? edge[(size_t)b * p.D + ch + j] : 0.f;
  if (p.flags) {
    const int group = step / G, first = group * G, before = step - first;
    const bool leader = before == G - 1 && step + 1 < p.nT;  // hands the group's end on
    if (w == 0 && !leader) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 m = joined(j);
        p.maps[((size_t)step * chains + chain) * C + lane * V + j] = m;
      }
      __threadfence();
      __syncwarp();
      if (lane == 0) store_release(p.flags + (size_t)step * chains + chain, 1);
    }
    if (w < before) {  // W >= G - 1: a warp fetches one earlier tile's map
      const size_t at = (size_t)(first + w) * chains + chain;
      wait_flag(p.flags + at);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 m = __ldcg(p.maps + at * C + lane * V + j);
        lP[w][lane * V + j] = m.x;
        lQ[w][lane * V + j] = m.y;
      }
    }
    float2 own[V];
#pragma unroll
    for (int j = 0; j < V; ++j) own[j] = leader && w == 0 ? joined(j) : make_float2(0.f, 0.f);
    __syncthreads();
    if (group > 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) c[j] = wait_end(p.ends + ((size_t)(group - 1) * chains + chain) * C + lane * V + j);
    }
#pragma unroll
    for (int i = 0; i < G - 1; ++i)
      if (i < before) {
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = through(lP[i][lane * V + j], lQ[i][lane * V + j], c[j]);
      }
    if (leader && w == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        put_end(p.ends + ((size_t)group * chains + chain) * C + lane * V + j, through(own[j].x, own[j].y, c[j]));
    }
  }
#pragma unroll
  for (int i = 0; i < W - 1; ++i)
    if (i < w) {
#pragma unroll
      for (int j = 0; j < V; ++j) c[j] = through(sP[i][lane * V + j], sQ[i][lane * V + j], c[j]);
    }

  // the rows, from the start value
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int t = row(r);
    if (t >= rows || !on) continue;
    const int at = t * p.D;
    bool first = !VAR && tile0 + t == 0, last = !VAR && tile0 + t == p.T - 1, out = false;
    int n = b;
    if (VAR) {
      const int code = sCode[t];
      first = code & ROW_START, last = code & ROW_END, out = code & ROW_OUT, n = code >> ROW_SHIFT;
      if (code & (ROW_OUT | (BWD ? ROW_END : ROW_START))) {
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = out || !edge ? 0.f : edge[(size_t)n * p.D + ch + j];
      }
    }
    PV y, z;
    if (!BWD) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        c[j] = out ? 0.f : fmaf(a[r][j], c[j], Num<T>::f(xv[r].v[j]));
        y.v[j] = Num<T>::t(c[j]);
      }
      *reinterpret_cast<PV *>(yp + at) = y;
      if (last && p.ht) {
#pragma unroll
        for (int j = 0; j < V; ++j) p.ht[(size_t)n * p.D + ch + j] = c[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float h = first ? (p.h0 ? p.h0[(size_t)n * p.D + ch + j] : 0.f) : Num<T>::f(ov[r].v[j]);
        const float d = out ? 0.f : Num<T>::f(xv[r].v[j]) + c[j];
        c[j] = out ? 0.f : a[r][j] * d;
        y.v[j] = Num<T>::t(d);
        z.v[j] = Num<T>::t(out ? 0.f : c[j] * h);
      }
      *reinterpret_cast<PV *>(yp + at) = y;
      *reinterpret_cast<PV *>(zp + at) = z;
      if (first && p.ht) {
#pragma unroll
        for (int j = 0; j < V; ++j) p.ht[(size_t)n * p.D + ch + j] = c[j];
      }
    }
  }
  // empty sequences hand their edge value through
  if (VAR && p.ht && step == 0 && on) {
    for (int n = w; n < p.N; n += W)
      if (cu_at(p, n) >= cu_at(p, n + 1)) {
#pragma unroll
        for (int j = 0; j < V; ++j) p.ht[(size_t)n * p.D + ch + j] = edge ? edge[(size_t)n * p.D + ch + j] : 0.f;
      }
  }
}

template <typename T> struct HgrnTile {
  static constexpr int W = 8, R = 16, L = W * R;
};

struct HgrnPlan {
  int V, C, nT, nCG;
  long long tiles;
  size_t flag_bytes, end_bytes, map_bytes;  // the first two are cleared before a launch
};

HgrnPlan hgrn_plan(int B, long long T, int D, int V, int L) {
  HgrnPlan q;
  q.V = V, q.C = 32 * V;
  q.nT = (int)((T + L - 1) / L);
  q.nCG = (D + q.C - 1) / q.C;
  q.tiles = (long long)q.nT * B * q.nCG;
  q.flag_bytes = ((size_t)(q.tiles + 1) * 4 + 255) / 256 * 256;
  q.map_bytes = (size_t)q.tiles * q.C * 8;
  q.end_bytes = (size_t)(q.nT / G) * B * q.nCG * q.C * 8;
  return q;
}

template <typename T, bool BWD, bool VAR, int V> int launch_hgrn(HgrnParams p, void *ws, size_t ws_bytes, cudaStream_t st) {
  typedef HgrnTile<T> G;
  const HgrnPlan q = hgrn_plan(p.B, p.T, p.D, V, G::L);
  p.nT = q.nT, p.nCG = q.nCG;
  FLAB_REQUIRE(q.tiles < (1ll << 31) && p.T < (1ll << 36) && p.D <= (1 << 23) && p.N < (1 << 28), FLAB_E_UNSUPPORTED,
               "hgrn: T = %lld, D = %d, N = %d are beyond what the kernel indexes", p.T, p.D, p.N);
  if (q.nT > 1) {
    FLAB_REQUIRE(ws && ws_bytes >= q.flag_bytes + q.map_bytes + q.end_bytes && reinterpret_cast<uintptr_t>(ws) % 16 == 0, FLAB_E_BADARG,
                 "hgrn needs a 16-byte aligned workspace of flab_hgrn_workspace() bytes");
    char *w = reinterpret_cast<char *>(ws);
    p.ticket = reinterpret_cast<int *>(w);
    p.flags = p.ticket + 1;
    p.ends = reinterpret_cast<unsigned long long *>(w + q.flag_bytes);
    p.maps = reinterpret_cast<float2 *>(w + q.flag_bytes + q.end_bytes);
    FLAB_REQUIRE(cudaMemsetAsync(w, 0, q.flag_bytes + q.end_bytes, st) == cudaSuccess, FLAB_E_LAUNCH, "hgrn: clearing the workspace failed");
  }
  hgrn_tile_kernel<T, V, G::W, G::R, BWD, VAR><<<(unsigned)q.tiles, G::W * 32, 0, st>>>(p);
  return check_launch(BWD ? "hgrn_bwd" : "hgrn_fwd");
}

template <typename T, bool BWD> int dispatch_hgrn(const HgrnParams &p, void *ws, size_t ws_bytes, cudaStream_t st) {
  constexpr int V = 2;
  bool vec = p.D % V == 0;
  for (const void *q : {p.x, p.g, p.o_in, (const void *)p.o, (const void *)p.dg}) vec = vec && reinterpret_cast<uintptr_t>(q) % (V * sizeof(T)) == 0;
  if (p.cu) return vec ? launch_hgrn<T, BWD, true, V>(p, ws, ws_bytes, st) : launch_hgrn<T, BWD, true, 1>(p, ws, ws_bytes, st);
  return vec ? launch_hgrn<T, BWD, false, V>(p, ws, ws_bytes, st) : launch_hgrn<T, BWD, false, 1>(p, ws, ws_bytes, st);
}

template <bool BWD> int run_hgrn(HgrnParams &p, int dtype, void *ws, size_t ws_bytes, cudaStream_t st) {
  switch (dtype) {
    case FLAB_BF16: return dispatch_hgrn<bf16, BWD>(p, ws, ws_bytes, st);
    case FLAB_FP16: return dispatch_hgrn<__half, BWD>(p, ws, ws_bytes, st);
    case FLAB_FP32: return dispatch_hgrn<float, BWD>(p, ws, ws_bytes, st);
    default: break;
  }
  set_error("hgrn: unknown dtype %d", dtype);
  return FLAB_E_BADARG;
}

}  // namespace
}  // namespace flab

extern "C" {

size_t flab_hgrn_workspace(int B, long long T, int D) {
  using namespace flab;
  if (B <= 0 || T <= 0 || D <= 0) return 0;
  size_t most = 0;  // of the layouts that a call of this size may take
  for (int V : {1, 2}) {
    const HgrnPlan q = hgrn_plan(B, T, D, V, HgrnTile<float>::L);
    const size_t n = q.nT > 1 ? q.flag_bytes + q.map_bytes + q.end_bytes : 0;
    most = n > most ? n : most;
  }
  return most;
}

int flab_hgrn_fwd(const void *x, const void *g, const float *h0, void *o, float *ht, const void *cu_seqlens, int cu_is_int64, int B, long long T,
                  int D, int N, int dtype, void *ws, size_t ws_bytes, void *stream) {
  using namespace flab;
  FLAB_REQUIRE(x && g && o && B > 0 && T > 0 && D > 0 && N > 0, FLAB_E_BADARG, "hgrn_fwd needs x, g, o and positive sizes");
  FLAB_REQUIRE(cu_seqlens ? B == 1 : N == B, FLAB_E_BADARG, "hgrn_fwd: packed sequences need B = 1, fixed-length batches N = B");
  HgrnParams p = {};
  p.x = x, p.g = g, p.h0 = h0, p.o = o, p.ht = ht, p.cu = cu_seqlens, p.cu64 = cu_is_int64;
  p.B = B, p.T = T, p.D = D, p.N = N;
  return run_hgrn<false>(p, dtype, ws, ws_bytes, (cudaStream_t)stream);
}

int flab_hgrn_bwd(const void *g, const void *o, const float *h0, const void *d_o, const float *dht, void *dx, void *dg, float *dh0,
                  const void *cu_seqlens, int cu_is_int64, int B, long long T, int D, int N, int dtype, void *ws, size_t ws_bytes, void *stream) {
  using namespace flab;
  FLAB_REQUIRE(g && o && d_o && dx && dg && B > 0 && T > 0 && D > 0 && N > 0, FLAB_E_BADARG, "hgrn_bwd needs g, o, do, dx, dg and positive sizes");
  FLAB_REQUIRE(cu_seqlens ? B == 1 : N == B, FLAB_E_BADARG, "hgrn_bwd: packed sequences need B = 1, fixed-length batches N = B");
  HgrnParams p = {};
  p.x = d_o, p.g = g, p.o_in = o, p.h0 = h0, p.dht = dht, p.o = dx, p.dg = dg, p.ht = dh0, p.cu = cu_seqlens, p.cu64 = cu_is_int64;
  p.B = B, p.T = T, p.D = D, p.N = N;
  return run_hgrn<true>(p, dtype, ws, ws_bytes, (cudaStream_t)stream);
}
}
