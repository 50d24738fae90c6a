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
// its group's earlier tiles.  The sums are formed in the same order whatever block runs when, so results repeat bit for bit (taking
// whichever of a predecessor's map and end value is there first does not repeat).  Groups of 4 and of 16 were slower (forward at
// [1, 262144, 1024] 480 and 575 us where groups of 8 took 344: more hops, and more maps to fetch).  Serial along time is one hop a group: a word
// of 64 bits that holds value and mark.  Tiles are handed out by a ticket in the order of time, so that a tile waits only for
// tiles whose blocks already run; one launch then reads everything once, where a two-pass scan would read the inputs twice.
// Three forms: rows that TMA can address stream through a persistent block (hgrn_stream_kernel), others go tile by tile through
// registers (hgrn_tile_kernel), and a few tokens a sequence are walked by one thread a channel group (hgrn_step_kernel).
// Measured against the bytes above at the copy rate of 6.55 TB/s, bf16: [8, 4096, 2048] forward 68 us (91 %), backward 107 us (96 %), in fp32
// 131 and 215 us with their launches (94 and 95 %); [1, 262144, 2048] forward 548 us (90 %), backward 872 us (94 %): 32 channel groups side
// by side, where a tile's wait for the maps of the tiles before it is what the stages no longer cover whole ([1, 262144, 1024] 310 and
// 480 us, 79 and 85 %; [1, 65536, 512] 55 and 83, 56 and 62 %); 64 packed sequences of 295926 tokens with their states 679 and 1044 us with
// the launches (82 and 89 %); one token of 256 x 2048 2.5 us.  Rows that TMA cannot address: [8, 4096, 2047] 267 and 288 us (23 and 36 %),
// loads of one element; the backward of that form spills 12 to 52 bytes a thread.
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
  int share;         // of the sequences, looked through for empty ones by each tile along time
  long long T;
  int *ticket;
  int *abort;                // set by a wait of this launch that ran out
  unsigned long long *maps;  // [tiles][C] words; null with one tile along time
  unsigned long long *ends;  // [groups][C] words
};

template <typename T, int V> struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack {
  T v[V];
};

// (held inside the tensor, whatever the caller's table says: it is never read on the host)
__device__ __forceinline__ long long cu_at(const HgrnParams &p, int n) {
  const long long v = p.cu64 ? reinterpret_cast<const long long *>(p.cu)[n] : (long long)reinterpret_cast<const int *>(p.cu)[n];
  return v < 0 ? 0 : v < p.T ? v : p.T;
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
// The factor of a map with factor `a` and one with factor `b` behind it.  A cut stays one: a product with it would make a NaN where gates
// above 1 have overflowed.  (Only sequences that are packed have cuts.)
template <bool VAR> __device__ __forceinline__ float behind(float a, float b) {
  return VAR && (int)(__float_as_uint(a) | __float_as_uint(b)) < 0 ? CUT : a * b;
}
// e^g as 2^(g log2 e): the product's rounding moves the result by |g| 2^-24 of itself, less than the exponential's own error
// wherever the gate is near 1 and errors live long.
__device__ __forceinline__ float gate(float g) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(g * 1.4426950408889634f));
  return y;
}

// The number of cumulative lengths that are <= t, by a warp together.
__device__ __forceinline__ int warp_count(const HgrnParams &p, long long t, int lane) {
  int lo = 0, hi = p.N + 1;
  while (lo < hi) {
    const int by = (hi - lo + 31) / 32, at = lo + lane * by;
    const int below = __popc(__ballot_sync(0xffffffffu, at < hi && cu_at(p, at) <= t));
    if (below == 0) break;
    hi = min(hi, lo + below * by);
    lo += (below - 1) * by + 1;
  }
  return lo;
}

// y = P c + Q.  A zero start stays out of the product, so that a P that overflowed (gates above 0) makes no NaN of it.
__device__ __forceinline__ float through(float P, float Q, float c) { return c == 0.f || is_cut(P) ? Q : fmaf(P, c, Q); }

// What tiles tell each other goes in words of 64 bits that hold a value and the mark that it is there, stored and loaded
// relaxed: whoever sees the mark has the value.  (A flag behind a fence was measured at 4000 cycles a tile under load.)  The
// words are cleared before the launch.
__device__ __forceinline__ unsigned long long end_word(float v) { return (1ull << 32) | __float_as_uint(v); }
__device__ __forceinline__ float end_of(unsigned long long w) { return __uint_as_float((unsigned)w); }
// A map: P's bits plus one are never 0 (the one pattern that would be, a NaN, is not what arithmetic makes of a NaN).
__device__ __forceinline__ unsigned long long map_word(float P, float Q) {
  return ((unsigned long long)(__float_as_uint(P) + 1u) << 32) | __float_as_uint(Q);
}
__device__ __forceinline__ float2 map_of(unsigned long long w) { return make_float2(__uint_as_float((unsigned)(w >> 32) - 1u), __uint_as_float((unsigned)w)); }
__device__ __forceinline__ void put(unsigned long long *a, unsigned long long w) {
  asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(a), "l"(w) : "memory");
}
__device__ __forceinline__ unsigned long long look(const unsigned long long *a) {
  unsigned long long w;
  asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(w) : "l"(a) : "memory");
  return w;
}
// What a wait that ran out hands back, as an end and as a map: NaN, so that nothing which depends on it looks like a result.
__device__ __forceinline__ unsigned long long lost() { return map_word(0.f, __uint_as_float(0x7fffffffu)); }
// Bounded wait for a word's mark, about a second; once any wait of the launch has run out, no further one of it waits.  (The error word
// is only written here: it stays set until the host clears it, and other launches are not to give up for it.  CALL: the record
// by a call.  Inlined, it costs the tile kernel registers ([8, 4096, 2047] bf16 forward 273 us against 265); the call costs the
// streaming kernel some ([1, 262144, 2048] forward 552 us against 547).)
__device__ __forceinline__ void give_up(int *abort) {
  *reinterpret_cast<volatile int *>(abort) = 1;
  tu_tc_error = 700;
}
__device__ __noinline__ void give_up_by_call(int *abort) { give_up(abort); }
template <bool CALL>
__device__ __forceinline__ unsigned long long await(const unsigned long long *a, unsigned long long w, int *abort, long long limit = 1ll << 31) {
  if (w >> 32) return w;
  const long long t0 = clock64();
  for (int spins = 1;; ++spins) {
    w = look(a);
    if (w >> 32) return w;
    if ((spins & 255) == 0 && (clock64() - t0 > limit || *reinterpret_cast<volatile int *>(abort))) {
      if (CALL) give_up_by_call(abort);
      else give_up(abort);
      return lost();
    }
  }
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
  if (p.maps) {
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
  bool cut = false;
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
        cut = true;
#pragma unroll
        for (int j = 0; j < V; ++j) Q[j] = (code & ROW_OUT) || !edge || !on ? 0.f : edge[(size_t)(code >> ROW_SHIFT) * p.D + ch + j];
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      a[r][j] = live ? gate(Num<T>::f(gv[r].v[j])) : 1.f;
      const float in = live ? Num<T>::f(xv[r].v[j]) : 0.f;
      Q[j] = BWD ? a[r][j] * (Q[j] + in) : fmaf(a[r][j], Q[j], in);
      P[j] *= a[r][j];
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) sP[w][lane * V + j] = VAR && cut ? CUT : P[j], sQ[w][lane * V + j] = Q[j];
  __syncthreads();

  auto joined = [&](int j) -> float2 {  // the tile's map of channel j of this lane
    float jP = 1.f, jQ = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float Pi = sP[i][lane * V + j];
      jQ = through(Pi, sQ[i][lane * V + j], jQ);
      jP = behind<VAR>(jP, Pi);
    }
    return make_float2(jP, jQ);
  };

  // the tile's start value: the end of the group of tiles before its own, taken through the maps of its group's earlier tiles
  float c[V];
#pragma unroll
  for (int j = 0; j < V; ++j) c[j] = !VAR && step < G && edge && on ? edge[(size_t)b * p.D + ch + j] : 0.f;
  if (p.maps) {
    const int group = step / G, first = group * G, before = step - first;
    const bool leader = before == G - 1 && step + 1 < p.nT;  // hands the group's end on
    if (w == 0 && !leader) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 m = joined(j);
        put(p.maps + ((size_t)step * chains + chain) * C + lane * V + j, map_word(m.x, m.y));
      }
    }
    if (w < before) {  // W >= G - 1: a warp fetches one earlier tile's map
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const unsigned long long *a = p.maps + ((size_t)(first + w) * chains + chain) * C + lane * V + j;
        const float2 m = map_of(await<true>(a, look(a), p.abort));
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
      for (int j = 0; j < V; ++j) {
        const unsigned long long *a = p.ends + ((size_t)(group - 1) * chains + chain) * C + lane * V + j;
        c[j] = end_of(await<true>(a, look(a), p.abort));
      }
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
        put(p.ends + ((size_t)group * chains + chain) * C + lane * V + j, end_word(through(own[j].x, own[j].y, c[j])));
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
  if (VAR && p.ht && on) {
    for (int n = step * p.share + w, to = min(step * p.share + p.share, p.N); n < to; n += W)
      if (cu_at(p, n) >= cu_at(p, n + 1)) {
#pragma unroll
        for (int j = 0; j < V; ++j) p.ht[(size_t)n * p.D + ch + j] = edge ? edge[(size_t)n * p.D + ch + j] : 0.f;
      }
  }
}

// ---- the streaming form: one persistent block an SM, tiles by TMA ----------------------------------------------------
// The same maps and order of sums, as a pipeline over S stages of shared memory whose warps meet only at mbarriers:
//   load warp    takes a ticket and fetches the tile (rows and channels outside the tensor arrive as zeros: the identity map)
//   map warps    compose the tile's rows, R to a warp, and wait for nothing outside the block
//   chain warps  publish the tile's map, fetch what came before it and leave the start value of every R rows
//   row warps    run the recurrence from there, outputs in place of inputs
//   store warp   sends the tile off and hands the stage back
// A tile's start value costs a trip or two to L2; the map warps being stages ahead of the row warps hides them, and keeps
// several groups of a long chain in flight.  Gates are evaluated twice (map, rows): two more instructions an element, against
// 64 registers a thread that would have to live through the wait.
template <typename T> __device__ __forceinline__ float2 unpack2(const T *s) {
  const Pack<T, 2> v = *reinterpret_cast<const Pack<T, 2> *>(s);
  return make_float2(Num<T>::f(v.v[0]), Num<T>::f(v.v[1]));
}
template <typename T> __device__ __forceinline__ void pack2(T *s, float a, float b) {
  Pack<T, 2> v;
  v.v[0] = Num<T>::t(a), v.v[1] = Num<T>::t(b);
  *reinterpret_cast<Pack<T, 2> *>(s) = v;
}
// The codes of the L rows from t0 on, by a warp: `n` is the last sequence that begins at or before t0 (-1: none).  Only the sequences
// that lie in the tile are looked at; a row between two edges has code 0.
template <int L> __device__ __forceinline__ void tile_codes(const HgrnParams &p, long long t0, int n, int *code, int lane) {
  const long long begin = cu_at(p, 0), end = cu_at(p, p.N);
  for (int r = lane; r < L; r += 32) code[r] = t0 + r < begin || t0 + r >= end ? ROW_OUT : 0;
  __syncwarp();
  for (int j0 = n < 0 ? 0 : n;; j0 += 32) {
    const int j = j0 + lane;
    bool inside = false;
    if (j < p.N) {
      const long long s = cu_at(p, j) - t0, e = cu_at(p, j + 1) - t0;  // first row, and the one behind the last
      inside = s < L;
      if (inside && s < e) {
        if (s >= 0) code[s] = (j << ROW_SHIFT) | ROW_START | (e == s + 1 ? ROW_END : 0);
        if (e > 0 && e <= L && e != s + 1) code[e - 1] = (j << ROW_SHIFT) | ROW_END;
      }
    }
    if (!__all_sync(0xffffffffu, inside)) break;
  }
}

// Empty sequences, where there are more of them than tokens: a warp each.
__global__ void __launch_bounds__(256) hgrn_empty_kernel(const HgrnParams p, const float *edge) {
  for (int n = blockIdx.x * 8 + (threadIdx.x >> 5); n < p.N; n += gridDim.x * 8)
    if (cu_at(p, n) >= cu_at(p, n + 1))
      for (int ch = threadIdx.x & 31; ch < p.D; ch += 32) p.ht[(size_t)n * p.D + ch] = edge ? edge[(size_t)n * p.D + ch] : 0.f;
}

// maps of two channels, one after the other (`a` first)
struct Map2 {
  float2 P, Q;
};
__device__ __forceinline__ float2 through(const Map2 &m, float2 c) { return make_float2(through(m.P.x, m.Q.x, c.x), through(m.P.y, m.Q.y, c.y)); }
template <bool VAR> __device__ __forceinline__ Map2 join(const Map2 &a, const Map2 &b) {
  Map2 m;
  m.Q = through(b, a.Q);
  m.P = make_float2(behind<VAR>(a.P.x, b.P.x), behind<VAR>(a.P.y, b.P.y));
  return m;
}

template <typename T, int R, int S, bool BWD> struct Stream {
  static constexpr int V = 2, C = 32 * V, W = 8, L = W * R;
  static constexpr int TILE = L * C, TENSORS = BWD ? 3 : 2;
  // One chain warp a stage: each sees every phase of its stage's barriers (a wait for a phase's parity says nothing to one that
  // has not seen the phase before it), and the waits of all stages overlap.
  static constexpr int CHAINS = S;
  static constexpr int THREADS = 32 * (2 * W + CHAINS + 2);
  struct Stage {
    T buf[TENSORS][TILE];   // x (do), g, o of a token earlier
    float2 P[W][32], Q[W][32];  // the warps' maps, then the maps of all rows before theirs
    float2 start[32];           // the tile's start value
    int code[L];
  };
  struct Shared {
    Stage st[S];
    struct Place {
      int step, chain, b, cg, t0, edges;  // step: position along the scan, -1 behind the last tile; edges: codes are set
    } at[S];
    uint64_t full[S], mapped[S], ready[S], done[S], empty[S];
  };
};

template <bool BWD, int L, int R> __device__ __forceinline__ int row_of(int w, int r) { return BWD ? L - 1 - (w * R + r) : w * R + r; }

template <typename T, int R, int S, bool BWD, bool VAR>
__global__ void __launch_bounds__(Stream<T, R, S, BWD>::THREADS, 1)
    hgrn_stream_kernel(const HgrnParams p, const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mg,
                       const __grid_constant__ CUtensorMap mo, const __grid_constant__ CUtensorMap my, const __grid_constant__ CUtensorMap mz) {
  typedef Stream<T, R, S, BWD> Z;
  constexpr int W = Z::W, L = Z::L, C = Z::C;
  constexpr int AHEAD = BWD ? ROW_END : ROW_START;  // the edge that a scan meets first
  extern __shared__ __align__(128) char raw[];
  typename Z::Shared &sh = *reinterpret_cast<typename Z::Shared *>(raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chains = p.B * p.nCG;
  const long long tiles = (long long)chains * p.nT;
  const float *const edge = BWD ? p.dht : p.h0;  // values in front of the sequences, in scan order
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      tc::mbar_init(&sh.full[s], 1);
      tc::mbar_init(&sh.mapped[s], W);
      tc::mbar_init(&sh.ready[s], 1);
      tc::mbar_init(&sh.done[s], W);
      tc::mbar_init(&sh.empty[s], 1);
    }
    tc::fence_barrier_init();
  }
  __syncthreads();
  // the codes of warp w's rows: bit r of the result where position r has one, lane r holds it
  auto codes_of = [&](int edges, const int *code, int w, int &mine) {
    mine = edges ? code[row_of<BWD, L, R>(w, lane % R)] : 0;
    return __ballot_sync(0xffffffffu, mine != 0) & (R == 32 ? ~0u : (1u << (R & 31)) - 1);
  };
  // position r of warp w's rows is this row of the tile
  auto row = [&](int w, int r) -> int { return row_of<BWD, L, R>(w, r); };

  if (warp < W) {  // ---- map warps
    const int w = warp;
    for (int it = 0;; ++it) {
      const int s = it % S;
      if (!tc::mbar_wait(&sh.full[s], (it / S) & 1)) {
        tu_tc_error = 702;
        break;
      }
      if (sh.at[s].step < 0) break;
      typename Z::Stage &st = sh.st[s];
      const T *const xs = st.buf[0] + lane * 2, *const gs = st.buf[1] + lane * 2;
      float2 P = make_float2(1.f, 1.f), Q = make_float2(0.f, 0.f);
      auto take = [&](float2 g, float2 x) {
        const float2 a = make_float2(gate(g.x), gate(g.y));
        Q.x = BWD ? a.x * (Q.x + x.x) : fmaf(a.x, Q.x, x.x);
        Q.y = BWD ? a.y * (Q.y + x.y) : fmaf(a.y, Q.y, x.y);
        P.x *= a.x, P.y *= a.y;
      };
      int mine = 0;
      const unsigned codes = VAR ? codes_of(sh.at[s].edges, st.code, w, mine) : 0;
      if (!VAR || codes == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) take(unpack2(gs + row(w, r) * C), unpack2(xs + row(w, r) * C));
      } else {
        // kept short: unrolled, this rarely run code cost more in instruction fetches than it saved
        const int ch = sh.at[s].cg * C + lane * 2;
        bool cut = false;
#pragma unroll 1
        for (int r = 0; r < R; ++r) {
          const float2 g = unpack2(gs + row(w, r) * C), x = unpack2(xs + row(w, r) * C);
          bool out = false;
          if (codes >> r & 1) {
            const int code = __shfl_sync(0xffffffffu, mine, r);
            out = code & ROW_OUT;
            if (code & (ROW_OUT | AHEAD)) {
              cut = true;
              Q = out || !edge || ch >= p.D ? make_float2(0.f, 0.f) : *reinterpret_cast<const float2 *>(edge + (size_t)(code >> ROW_SHIFT) * p.D + ch);
            }
          }
          if (!out) take(g, x);
        }
        if (cut) P = make_float2(CUT, CUT);
      }
      st.P[w][lane] = P;
      st.Q[w][lane] = Q;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sh.mapped[s]);
    }
  } else if (warp < 2 * W) {  // ---- row warps
    const int w = warp - W;
    for (int it = 0;; ++it) {
      const int s = it % S;
      if (!tc::mbar_wait(&sh.full[s], (it / S) & 1)) {
        tu_tc_error = 703;
        break;
      }
      if (sh.at[s].step < 0) break;
      if (!tc::mbar_wait(&sh.ready[s], (it / S) & 1)) {
        tu_tc_error = 704;
        break;
      }
      typename Z::Stage &st = sh.st[s];
      const typename Z::Shared::Place z = sh.at[s];
      const int ch = z.cg * C + lane * 2;
      const bool on = ch < p.D;
      T *const xs = st.buf[0] + lane * 2, *const gs = st.buf[1] + lane * 2;
      const T *const os = st.buf[BWD ? 2 : 0] + lane * 2;
      float2 c = st.start[lane];
      if (w > 0) c = make_float2(through(st.P[w][lane].x, st.Q[w][lane].x, c.x), through(st.P[w][lane].y, st.Q[w][lane].y, c.y));
      auto take = [&](int at, float2 g, float2 x, float2 h) {
        const float2 a = make_float2(gate(g.x), gate(g.y));
        if (!BWD) {
          c.x = fmaf(a.x, c.x, x.x), c.y = fmaf(a.y, c.y, x.y);
          pack2(xs + at, c.x, c.y);
        } else {
          const float2 d = make_float2(x.x + c.x, x.y + c.y);
          c.x = a.x * d.x, c.y = a.y * d.y;
          pack2(xs + at, d.x, d.y);
          pack2(gs + at, c.x * h.x, c.y * h.y);
        }
      };
      const float2 none = make_float2(0.f, 0.f);
      int mine = 0;
      const unsigned codes = VAR ? codes_of(z.edges, st.code, w, mine) : 0;
      if (!VAR || codes == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int at = row(w, r) * C;
          float2 h = BWD ? unpack2(os + at) : none;
          // the first token's h_{t-1} (the load of it fell in front of the tensor and arrived as 0)
          if (BWD && !VAR && r == R - 1 && w == W - 1 && z.t0 == 0 && p.h0 && on) h = *reinterpret_cast<const float2 *>(p.h0 + (size_t)z.b * p.D + ch);
          take(at, unpack2(gs + at), unpack2(xs + at), h);
        }
      } else {
#pragma unroll 1
        for (int r = 0; r < R; ++r) {
          const int at = row(w, r) * C;
          const float2 g = unpack2(gs + at), x = unpack2(xs + at);
          float2 h = BWD ? unpack2(os + at) : none;
          int code = 0;
          if (codes >> r & 1) {
            code = __shfl_sync(0xffffffffu, mine, r);
            const size_t of = (size_t)(code >> ROW_SHIFT) * p.D + ch;
            if (code & AHEAD) c = edge && on ? *reinterpret_cast<const float2 *>(edge + of) : none;
            if (BWD && (code & ROW_START)) h = p.h0 && on ? *reinterpret_cast<const float2 *>(p.h0 + of) : none;
          }
          if (code & ROW_OUT) {
            c = none;
            pack2(xs + at, 0.f, 0.f);
            if (BWD) pack2(gs + at, 0.f, 0.f);
          } else {
            take(at, g, x, h);
            if ((code & (BWD ? ROW_START : ROW_END)) && p.ht && on) *reinterpret_cast<float2 *>(p.ht + (size_t)(code >> ROW_SHIFT) * p.D + ch) = c;
          }
        }
      }
      // rows past T are the identity, so the last warp's last value is the sequence's
      if (!VAR && z.step == p.nT - 1 && w == W - 1 && p.ht && on) *reinterpret_cast<float2 *>(p.ht + (size_t)z.b * p.D + ch) = c;
      if (VAR && p.ht && on) {  // empty sequences hand their edge value through
        for (int n = z.step * p.share + w, to = min(z.step * p.share + p.share, p.N); n < to; n += W)
          if (cu_at(p, n) >= cu_at(p, n + 1))
            *reinterpret_cast<float2 *>(p.ht + (size_t)n * p.D + ch) = edge ? *reinterpret_cast<const float2 *>(edge + (size_t)n * p.D + ch) : none;
      }
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sh.done[s]);
    }
  } else if (warp < 2 * W + Z::CHAINS) {  // ---- chain warps
    for (int it = warp - 2 * W;; it += Z::CHAINS) {
      const int s = it % S;
      if (!tc::mbar_wait(&sh.full[s], (it / S) & 1)) {
        tu_tc_error = 705;
        break;
      }
      if (sh.at[s].step < 0) break;
      if (!tc::mbar_wait(&sh.mapped[s], (it / S) & 1)) {
        tu_tc_error = 706;
        break;
      }
      typename Z::Stage &st = sh.st[s];
      const typename Z::Shared::Place z = sh.at[s];
      const int ch = z.cg * C + lane * 2;
      const int group = z.step / G, first = group * G, before = z.step - first;
      const bool leader = before == G - 1 && z.step + 1 < p.nT;  // hands the group's end on
      auto words = [&](unsigned long long *base, int step) { return base + ((size_t)step * chains + z.chain) * C + lane * 2; };
      auto rows_map = [&](int i) {
        Map2 m;
        m.P = st.P[i][lane], m.Q = st.Q[i][lane];
        return m;
      };
      // the tile's map, by halves: what other tiles wait for goes out first
      const Map2 tile = join<VAR>(join<VAR>(join<VAR>(rows_map(0), rows_map(1)), join<VAR>(rows_map(2), rows_map(3))),
                                  join<VAR>(join<VAR>(rows_map(4), rows_map(5)), join<VAR>(rows_map(6), rows_map(7))));
      if (before < G - 1 && z.step + 1 < p.nT) {
        put(words(p.maps, z.step), map_word(tile.P.x, tile.Q.x));
        put(words(p.maps, z.step) + 1, map_word(tile.P.y, tile.Q.y));
      }
      // everything that comes before is asked for at once; the earlier tiles of the group again and again until all of them are there,
      // and then the end of the group before, which is last to come where tiles wait at all
      unsigned long long g[G - 1][2], e[2] = {0, 0};
      const unsigned long long *const maps = words(p.maps, first), *const ends = words(p.ends, group > 0 ? group - 1 : 0);
      const size_t by = (size_t)chains * C;
#pragma unroll
      for (int i = 0; i < G - 1; ++i)
        if (i < before) g[i][0] = look(maps + i * by), g[i][1] = look(maps + i * by + 1);
      if (group > 0) e[0] = look(ends), e[1] = look(ends + 1);
      {  // meanwhile, the way from the tile's start to each warp's rows takes the place of the rows' own map
        Map2 to = rows_map(0);
#pragma unroll
        for (int i = 1; i < W; ++i) {
          const Map2 own = rows_map(i);
          st.P[i][lane] = to.P, st.Q[i][lane] = to.Q;
          if (i + 1 < W) to = join<VAR>(to, own);
        }
      }
      const long long asked = clock64();
      for (int spins = 1;; ++spins) {
        bool missing = false;
#pragma unroll
        for (int i = 0; i < G - 1; ++i) missing = missing || (i < before && !((g[i][0] >> 32) && (g[i][1] >> 32)));
        if (!__any_sync(0xffffffffu, missing)) break;
        // the wait has a bound like every other: about a second, and none once any of the launch has run out
        if ((spins & 255) == 0 && __any_sync(0xffffffffu, clock64() - asked > (1ll << 31) || *reinterpret_cast<volatile int *>(p.abort))) {
          give_up(p.abort);
#pragma unroll
          for (int i = 0; i < G - 1; ++i)
            for (int k = 0; k < 2; ++k)
              if (!(g[i][k] >> 32)) g[i][k] = lost();
          break;
        }
#pragma unroll
        for (int i = 0; i < G - 1; ++i)
          if (i < before) {
            if (!(g[i][0] >> 32)) g[i][0] = look(maps + i * by);
            if (!(g[i][1] >> 32)) g[i][1] = look(maps + i * by + 1);
          }
        if (group > 0) {
          if (!(e[0] >> 32)) e[0] = look(ends);
          if (!(e[1] >> 32)) e[1] = look(ends + 1);
        }
      }
      // the group's earlier tiles as one map, then its start
      auto tile_map = [&](int i) {
        const float2 x = map_of(g[i][0]), y = map_of(g[i][1]);
        Map2 m;
        m.P = i < before ? make_float2(x.x, y.x) : make_float2(1.f, 1.f);
        m.Q = i < before ? make_float2(x.y, y.y) : make_float2(0.f, 0.f);
        return m;
      };
      const Map2 group_map = join<VAR>(join<VAR>(join<VAR>(tile_map(0), tile_map(1)), join<VAR>(tile_map(2), tile_map(3))),
                                       join<VAR>(join<VAR>(tile_map(4), tile_map(5)), tile_map(6)));
      float2 c = make_float2(0.f, 0.f);
      if (group > 0) {
        c = make_float2(end_of(await<false>(ends, e[0], p.abort)), end_of(await<false>(ends + 1, e[1], p.abort)));
      }
      else if (!VAR && edge && ch < p.D) c = *reinterpret_cast<const float2 *>(edge + (size_t)z.b * p.D + ch);
      c = through(group_map, c);
      if (leader) {
        const float2 end = through(tile, c);
        put(words(p.ends, group), end_word(end.x));
        put(words(p.ends, group) + 1, end_word(end.y));
      }
      st.start[lane] = c;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&sh.ready[s]);
    }
  } else if (warp == 2 * W + Z::CHAINS) {  // ---- load warp
    int tile = 0, first_seq = BWD ? p.N : 0;  // the last sequence that begins at or before the tile (packed batches)
    if (lane == 0) tile = atomicAdd(p.ticket, 1);
    tile = __shfl_sync(0xffffffffu, tile, 0);
    for (int it = 0;; ++it) {
      const int s = it % S;
      // what the tile's place takes (and the next ticket) falls into the wait for the stage
      const bool more = tile < tiles;
      typename Z::Shared::Place z;
      z.step = -1;
      int following = 0;
      if (more) {
        if (lane == 0) following = atomicAdd(p.ticket, 1);
        z.step = tile / chains;
        z.chain = tile - z.step * chains;
        z.b = z.chain / p.nCG;
        z.cg = z.chain - z.b * p.nCG;
        z.t0 = (BWD ? p.nT - 1 - z.step : z.step) * L;
        z.edges = 0;
        if (VAR) {  // most tiles lie inside one sequence
          // tickets go along time: the sequence is found among the 32 next to the last tile's, with one load
          const int from = max(BWD ? first_seq - 30 : first_seq, 0);
          const long long v = cu_at(p, min(from + lane, p.N));
          const int below = __popc(__ballot_sync(0xffffffffu, from + lane <= p.N && v <= z.t0));
          if ((below > 0 || from == 0) && below < 32) {
            first_seq = from + below - 1;
            const long long b0 = __shfl_sync(0xffffffffu, v, max(below - 1, 0)), b1 = __shfl_sync(0xffffffffu, v, below);
            z.edges = first_seq < 0 || first_seq >= p.N || b0 == z.t0 || b1 <= z.t0 + L;
          } else {
            first_seq = warp_count(p, z.t0, lane) - 1;
            z.edges = first_seq < 0 || first_seq >= p.N || cu_at(p, first_seq) == z.t0 || cu_at(p, first_seq + 1) <= z.t0 + L;
          }
        }
      }
      if (it >= S && !tc::mbar_wait(&sh.empty[s], (it / S - 1) & 1)) {
        tu_tc_error = 707;
        break;
      }
      __syncwarp();
      if (more) {
        typename Z::Stage &st = sh.st[s];
        if (lane == 0) {
          tc::tma_load_3d(st.buf[1], &mg, &sh.full[s], z.cg * C, z.t0, z.b);
          tc::tma_load_3d(st.buf[0], &mx, &sh.full[s], z.cg * C, z.t0, z.b);
          if (BWD) tc::tma_load_3d(st.buf[Z::TENSORS - 1], &mo, &sh.full[s], z.cg * C, z.t0 - 1, z.b);
        }
        if (VAR && z.edges) tile_codes<L>(p, z.t0, first_seq, st.code, lane);
      }
      __syncwarp();
      if (lane == 0) {
        sh.at[s] = z;
        if (more) tc::mbar_expect_tx(&sh.full[s], Z::TENSORS * Z::TILE * sizeof(T));
        else tc::mbar_arrive(&sh.full[s]);
      }
      // every chain warp is told of the end in its own next stage
      if (!more) {
        for (int next = it + 1; next < it + Z::CHAINS; ++next) {
          const int n = next % S;
          if (next >= S && !tc::mbar_wait(&sh.empty[n], (next / S - 1) & 1)) {
            tu_tc_error = 708;
            break;
          }
          if (lane == 0) {
            sh.at[n].step = -1;
            tc::mbar_arrive(&sh.full[n]);
          }
        }
        break;
      }
      tile = __shfl_sync(0xffffffffu, following, 0);
    }
  } else if (lane == 0) {  // ---- store warp
    for (int it = 0;; ++it) {
      const int s = it % S;
      if (!tc::mbar_wait(&sh.full[s], (it / S) & 1)) {
        tu_tc_error = 709;
        break;
      }
      if (sh.at[s].step < 0) break;
      if (!tc::mbar_wait(&sh.done[s], (it / S) & 1)) {
        tu_tc_error = 710;
        break;
      }
      const typename Z::Shared::Place z = sh.at[s];
      tc::tma_store_3d(&my, sh.st[s].buf[0], z.cg * C, z.t0, z.b);
      if (BWD) tc::tma_store_3d(&mz, sh.st[s].buf[1], z.cg * C, z.t0, z.b);
      tc::tma_store_commit();
      tc::tma_store_wait_read();
      tc::mbar_arrive(&sh.empty[s]);
    }
    tc::tma_store_wait_all();
  }
  __syncthreads();
}

// ---- a few tokens a sequence (decode, short windows) --------------------------------------------------------------------
// A thread walks the tokens of its channels; nothing is shared.
template <typename T, int V, bool BWD> __global__ void __launch_bounds__(256) hgrn_step_kernel(const HgrnParams p) {
  const int per = p.D / V;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)p.B * per) return;
  const int b = (int)(i / per), ch = (int)(i - (long long)b * per) * V;
  const float *const edge = BWD ? p.dht : p.h0;
  typedef Pack<T, V> PV;
  typedef Pack<float, V> PF;
  PF c, h;
#pragma unroll
  for (int j = 0; j < V; ++j) c.v[j] = h.v[j] = 0.f;
  const size_t state = (size_t)b * p.D + ch;
  if (edge) c = *reinterpret_cast<const PF *>(edge + state);
  if (BWD && p.h0) h = *reinterpret_cast<const PF *>(p.h0 + state);
  constexpr int U = BWD && V * sizeof(T) == 16 ? 4 : 8;  // tokens whose loads are in flight together
  const int last = (int)p.T - 1;
  for (int k0 = 0; k0 <= last; k0 += U) {
    PV g[U], x[U], o[BWD ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u <= last) {
        const int t = BWD ? last - (k0 + u) : k0 + u;
        const size_t at = ((size_t)b * p.T + t) * p.D + ch;
        g[u] = *reinterpret_cast<const PV *>(reinterpret_cast<const T *>(p.g) + at);
        x[u] = *reinterpret_cast<const PV *>(reinterpret_cast<const T *>(p.x) + at);
        if (BWD && t > 0) o[u] = *reinterpret_cast<const PV *>(reinterpret_cast<const T *>(p.o_in) + at - p.D);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u <= last) {
        const int t = BWD ? last - (k0 + u) : k0 + u;
        const size_t at = ((size_t)b * p.T + t) * p.D + ch;
        PV y, z;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float a = gate(Num<T>::f(g[u].v[j]));
          if (!BWD) {
            c.v[j] = fmaf(a, c.v[j], Num<T>::f(x[u].v[j]));
            y.v[j] = Num<T>::t(c.v[j]);
          } else {
            const float d = Num<T>::f(x[u].v[j]) + c.v[j];
            c.v[j] = a * d;
            y.v[j] = Num<T>::t(d);
            z.v[j] = Num<T>::t(c.v[j] * (t > 0 ? Num<T>::f(o[BWD ? u : 0].v[j]) : h.v[j]));
          }
        }
        *reinterpret_cast<PV *>(reinterpret_cast<T *>(p.o) + at) = y;
        if (BWD) *reinterpret_cast<PV *>(reinterpret_cast<T *>(p.dg) + at) = z;
      }
  }
  if (p.ht) *reinterpret_cast<PF *>(p.ht + state) = c;
}

// A wait that is meant to run out, on a word that nothing sets.  status[32] is its call's abort flag.
__device__ unsigned long long never_set = 0;
__global__ void __launch_bounds__(32) hgrn_wait_selftest_kernel(long long limit_ticks, int *status) {
  const unsigned long long w = await<false>(&never_set, look(&never_set), status + 32, limit_ticks);
  if (threadIdx.x == 0) *status = isnan(end_of(w)) && isnan(map_of(w).y) ? 700 : 0;
}

template <typename T> struct HgrnTile {
  static constexpr int W = 8, R = 16, L = W * R;
};

struct HgrnPlan {
  int V, C, nT, nCG;
  long long tiles;
  size_t bytes, end_bytes, map_bytes;  // the ticket and the abort flag (256 bytes), the ends, the maps
};

HgrnPlan hgrn_plan(int B, long long T, int D, int V, int L) {
  HgrnPlan q;
  q.V = V, q.C = 32 * V;
  q.nT = (int)((T + L - 1) / L);
  q.nCG = (D + q.C - 1) / q.C;
  q.tiles = (long long)q.nT * B * q.nCG;
  q.map_bytes = q.nT > 1 ? (size_t)q.tiles * q.C * 8 : 0;
  q.end_bytes = (size_t)(q.nT / G) * B * q.nCG * q.C * 8;
  q.bytes = 256 + q.end_bytes + q.map_bytes;
  return q;
}

// Hands the workspace out and clears it.
int hgrn_scratch(HgrnParams &p, const HgrnPlan &q, void *ws, size_t ws_bytes, cudaStream_t st) {
  FLAB_REQUIRE(ws && ws_bytes >= q.bytes && reinterpret_cast<uintptr_t>(ws) % 16 == 0, FLAB_E_BADARG,
               "hgrn needs a 16-byte aligned workspace of flab_hgrn_workspace() bytes");
  char *w = reinterpret_cast<char *>(ws);
  p.ticket = reinterpret_cast<int *>(w);
  p.abort = p.ticket + 32;
  p.ends = reinterpret_cast<unsigned long long *>(w + 256);
  p.maps = reinterpret_cast<unsigned long long *>(w + 256 + q.end_bytes);
  FLAB_REQUIRE(cudaMemsetAsync(w, 0, q.bytes, st) == cudaSuccess, FLAB_E_LAUNCH, "hgrn: clearing the workspace failed");
  return FLAB_OK;
}

// Which sequences the tiles look through.  One by one they take a tile's warps 0.1 us each (4 million by a single tile 350 ms, and a wait
// that runs out is not far), so every tile along time takes a share; and where that is more than two a token, so that most are
// empty, a kernel of their own looks through all.
int share_of(const HgrnParams &p, int L) {
  const long long share = ((long long)p.N + p.nT - 1) / p.nT;
  return !p.ht || share > 2 * L ? 0 : (int)share;
}
template <bool BWD> int pass_empty(const HgrnParams &p, cudaStream_t st) {
  if (!p.cu || !p.ht || p.share) return FLAB_OK;
  const long long blocks = ((long long)p.N + 7) / 8, most = sm_count() * 8ll;
  hgrn_empty_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>(p, BWD ? p.dht : p.h0);
  return check_launch(BWD ? "hgrn_bwd" : "hgrn_fwd");
}

template <typename T, bool BWD, bool VAR, int V> int launch_hgrn(HgrnParams p, void *ws, size_t ws_bytes, cudaStream_t st) {
  typedef HgrnTile<T> Z;
  const HgrnPlan q = hgrn_plan(p.B, p.T, p.D, V, Z::L);
  p.nT = q.nT, p.nCG = q.nCG;
  if (q.nT > 1) {
    const int rc = hgrn_scratch(p, q, ws, ws_bytes, st);
    if (rc) return rc;
  }
  p.share = share_of(p, Z::L);
  hgrn_tile_kernel<T, V, Z::W, Z::R, BWD, VAR><<<(unsigned)q.tiles, Z::W * 32, 0, st>>>(p);
  const int rc = check_launch(BWD ? "hgrn_bwd" : "hgrn_fwd");
  return rc ? rc : pass_empty<BWD>(p, st);
}

template <typename T, bool BWD> struct StreamOf {  // 32 KB (48 KB) of inputs a stage, as many stages as an SM holds
  static constexpr int R = sizeof(T) == 2 ? 16 : 8, S = BWD ? 4 : 6;
};

template <typename T, bool BWD, bool VAR, int R = StreamOf<T, BWD>::R, int S = StreamOf<T, BWD>::S>
int launch_stream(HgrnParams p, void *ws, size_t ws_bytes, cudaStream_t st) {
  typedef Stream<T, R, S, BWD> Z;
  const HgrnPlan q = hgrn_plan(p.B, p.T, p.D, Z::V, Z::L);
  p.nT = q.nT, p.nCG = q.nCG;
  int rc = hgrn_scratch(p, q, ws, ws_bytes, st);
  if (rc) return rc;
  const CUtensorMapDataType type = sizeof(T) == 4                ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : Num<T>::id == FLAB_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t dims[3] = {(uint64_t)p.D, (uint64_t)p.T, (uint64_t)p.B};
  const uint64_t strides[2] = {(uint64_t)p.D * sizeof(T), (uint64_t)p.T * p.D * sizeof(T)};
  const uint32_t box[3] = {Z::C, Z::L, 1};
  CUtensorMap m[5];
  const void *base[5] = {p.x, p.g, BWD ? p.o_in : p.x, p.o, BWD ? p.dg : p.o};
  for (int i = 0; i < 5; ++i)
    if ((rc = make_tensor_map(&m[i], base[i], type, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B))) return rc;
  auto kernel = hgrn_stream_kernel<T, R, S, BWD, VAR>;
  const int bytes = (int)sizeof(typename Z::Shared);
  if ((rc = set_smem(kernel, bytes))) return rc;
  const int sms = sm_count();
  const long long grid = q.tiles < sms ? q.tiles : sms;
  p.share = share_of(p, Z::L);
  kernel<<<(unsigned)grid, Z::THREADS, bytes, st>>>(p, m[0], m[1], m[2], m[3], m[4]);
  rc = check_launch(BWD ? "hgrn_bwd" : "hgrn_fwd");
  return rc ? rc : pass_empty<BWD>(p, st);
}

// Fixed-length sequences of up to WALK tokens are walked by one thread a channel group instead of being put into tiles, which they
// would leave mostly empty.  Rows that TMA cannot address are walked up to a tile's 128 tokens where the channels alone fill the card.
constexpr int WALK = 32;
bool walks(const HgrnParams &p, int V, bool tma) {
  return !p.cu && (p.T <= WALK || (!tma && p.T <= 128 && (long long)p.B * p.D / V >= 512ll * sm_count()));
}

template <typename T, bool BWD, int V> int launch_step(const HgrnParams &p, cudaStream_t st) {
  const long long n = (long long)p.B * (p.D / V);
  hgrn_step_kernel<T, V, BWD><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p);
  return check_launch(BWD ? "hgrn_bwd" : "hgrn_fwd");
}

template <typename T, bool BWD> int dispatch_hgrn(const HgrnParams &p, void *ws, size_t ws_bytes, cudaStream_t st) {
  FLAB_REQUIRE(p.T < (1ll << 30) && p.D <= (1 << 23) && p.N < (1 << 28) && (p.T + 63) / 64 * p.B * ((p.D + 31) / 32) < (1ll << 31), FLAB_E_UNSUPPORTED,
               "hgrn: B = %d, T = %lld, D = %d, N = %d are beyond what the kernels index", p.B, p.T, p.D, p.N);
  bool pair = p.D % 2 == 0, tma = p.D * sizeof(T) % 16 == 0;
  for (const void *q : {p.x, p.g, p.o_in, (const void *)p.o, (const void *)p.dg}) {
    pair = pair && reinterpret_cast<uintptr_t>(q) % (2 * sizeof(T)) == 0;
    tma = tma && reinterpret_cast<uintptr_t>(q) % 16 == 0;
  }
  for (const float *q : {p.h0, p.dht, (const float *)p.ht}) tma = tma && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  // The streaming form walks all sequences that lie in a tile, 32 in half a microsecond, and all of the table may lie in one (empty ones):
  // some 50 ms for 4 million, of the second that a wait bears.  Larger tables go by the tile form, which searches for each row's sequence:
  // 2 million sequences of two tokens, 64 channels, take it 5.3 ms where the streaming form takes 2.7.  (Past runs of empty ones in steps
  // that double, the code that does it cost every packed call 2 %.)
  if (p.cu && p.N > 1 << 22) tma = false;
  constexpr int WIDE = 16 / sizeof(T);
  bool wide = tma && p.D % WIDE == 0;
  for (const float *q : {p.h0, p.dht, (const float *)p.ht}) {
    wide = wide && reinterpret_cast<uintptr_t>(q) % 16 == 0;
    pair = pair && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  }
  if (walks(p, wide ? WIDE : pair ? 2 : 1, tma))
    return wide ? launch_step<T, BWD, WIDE>(p, st) : pair ? launch_step<T, BWD, 2>(p, st) : launch_step<T, BWD, 1>(p, st);
  if constexpr (!BWD && sizeof(T) == 2) {
    // Long sequences with few channel groups side by side: tiles of twice the rows, and half the hops along time.  Forward, bf16, 128
    // against 256 rows a tile: [1, 16384, 512] 22.7 -> 18.2 us, [1, 8192, 1024] 18.8 -> 17.8, [1, 65536, 512] 69 -> 55, [1, 262144, 2048]
    // 569 -> 550, [4, 65536, 2048] 536 -> 515; and the other way [1, 16384, 2048] 45.7 -> 47.8, [4, 4096, 2048] 46.0 -> 47.4, and
    // packed sequences of 290000 tokens 660 -> 699.
    const long long groups = (long long)p.B * ((p.D + 63) / 64);
    if (tma && !p.cu && (groups <= 16 ? p.T >= 8192 : groups <= 128 && p.T >= 32768)) return launch_stream<T, BWD, false, 32, 3>(p, ws, ws_bytes, st);
  }
  if (tma)
    return p.cu ? launch_stream<T, BWD, true>(p, ws, ws_bytes, st) : launch_stream<T, BWD, false>(p, ws, ws_bytes, st);
  if (p.cu) return pair ? launch_hgrn<T, BWD, true, 2>(p, ws, ws_bytes, st) : launch_hgrn<T, BWD, true, 1>(p, ws, ws_bytes, st);
  return pair ? launch_hgrn<T, BWD, false, 2>(p, ws, ws_bytes, st) : launch_hgrn<T, BWD, false, 1>(p, ws, ws_bytes, st);
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
  if (B <= 0 || T <= 0 || D <= 0 || (B > 1 && T <= WALK)) return 0;
  size_t most = 0;  // of the layouts that a call of this size may take
  for (int V : {1, 2})
    for (int L : {64, HgrnTile<float>::L}) {
      const HgrnPlan q = hgrn_plan(B, T, D, V, L);
      const size_t n = q.bytes;
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

int flab_hgrn_wait_selftest(long long limit_ticks, int *status, void *stream) {
  using namespace flab;
  FLAB_REQUIRE(status != nullptr, FLAB_E_BADARG, "hgrn_wait_selftest: NULL status");
  FLAB_REQUIRE(limit_ticks > 0 && limit_ticks <= (1ll << 28), FLAB_E_BADARG,
               "hgrn_wait_selftest: the limit must be between 1 and 2^28 clock ticks (a fraction of a second)");
  hgrn_wait_selftest_kernel<<<1, 32, 0, (cudaStream_t)stream>>>(limit_ticks, status);
  return check_launch("hgrn_wait_selftest");
}
}
