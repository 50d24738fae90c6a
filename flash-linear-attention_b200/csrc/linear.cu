// Products with an epilogue, for the projections either side of the recurrences (nn.Linear in fla/layers; the epilogue's parts are
// separate PyTorch kernels there):
//   y = act(x W^T + b) + r            x [M, K], W [N, K] bf16 / fp16, or e4m3 bytes with a scale a row of each
//   backward:  dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum over rows of dz;  dr = dy
// One tcgen05 kernel computes all three products, C[m, n] = sum_k A(m, k) B(n, k), with either operand stored row by row
// (K-major) or column by column (MN-major: W in dx, dz and x in dW), so nothing is transposed in memory.  Accumulation fp32 in TMEM;
// the epilogue is fp32 and rounds once.  z is kept for backward in the type of x, and dz is rounded to that type because it is an operand
// of both products.  The rounding of z moves a slope by up to |act''| |z| eps / 2: below dz's own rounding where the slope is near 1,
// above it where the slope is small (in the tails of the two sigmoids |z| times it, 8 times at z = 8; near a zero of silu's or gelu's slope
// without bound, relative to it).  It halves the bytes of what is kept; gradients are 2.4e-3 off the 64-bit ones where fp32 would give 1.7e-3.
//
// Layout: a pair of CTAs works on a 256 x BN tile (cta_group::2), each CTA loading its 128 rows of A and its half of B, S stages of
// 128-byte rows by TMA; the accumulator is double buffered in TMEM so that a tile's epilogue runs under the next tile's products.
// An epilogue thread holds a row of the accumulator; its results go through swizzled shared memory to TMA tile stores, and the
// residual comes in the same way, a block ahead.  Outputs whose rows do not begin on 16-byte boundaries go through a transposition in
// shared memory instead, so that a warp reads and writes runs of 64 bytes.  Tiles go in groups of 8 rows of tiles, so that what the
// pairs work on at one time shares operands in L2.
// Measured, bf16, 32768 x 2048 x 2048: product alone 183 us (1499 TFLOP/s; the library's 179), with silu, bias and residual 194 us, dx
// 181, dW 185 us (the library's 179); 8192 x 8192 x 8192 706 to 736 us by card (the library's 649 to 663), dx 858 to 870, dW 860 (757 to
// 815).  e4m3, 32768 x 2048 x 2048 with scales 105 to 108 us, with silu 121 to 135.  Bound by the tensor pipe under the power cap (88 to
// 93 % active without an epilogue, 83 % with one).  256 x 2048 x 2048 takes 12.0 us (the library's 5.1): one row of tiles, so 64 of 148
// SMs, each bound by what it can take in from L2; 16 x 2048 x 8192 16.4 us (5.6), where most of a tile is rows that are not there.
// The forward epilogue without tile stores spills 52 to 136 bytes a thread.
#include <type_traits>

#include "tc.cuh"

FLAB_TC_DEFINE_ERROR_WORD(linear_error)

namespace flab {
namespace {

enum { ACT_NONE = 0, ACT_SILU = 1, ACT_SIGMOID = 2, ACT_LOGSIGMOID = 3, ACT_GELU = 4 };

// 1 / (1 + e^-z) from the hardware's base-2 exponential and reciprocal (about 2^-22 of the value; e^-z beyond fp32 gives 0 as it should)
__device__ __forceinline__ float sigmoid(float z) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}
__device__ __forceinline__ float act_fwd(float z, int act) {
  switch (act) {
    case ACT_SILU: return z * sigmoid(z);
    case ACT_SIGMOID: return sigmoid(z);
    case ACT_LOGSIGMOID: return fminf(z, 0.f) - log1pf(__expf(-fabsf(z)));
    case ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    default: return z;
  }
}
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case ACT_SILU: {
      const float s = sigmoid(z);
      return fmaf(z, fmaf(-s, s, s), s);
    }
    case ACT_SIGMOID: {  // e / (1 + e)^2 with e = e^-|z|: s - s^2 would cancel where s is near 1
      float e, s;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fabsf(z) * -1.4426950408889634f));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
      return e * s * s;
    }
    case ACT_LOGSIGMOID: return sigmoid(-z);
    case ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * __expf(-0.5f * z * z);
    default: return 1.f;
  }
}

// z as it is kept for backward: held at the type's largest number where fp32 holds it and fp16 does not. The slopes are flat out there,
// and an infinity would make a product 0 * inf of them. What is not finite in fp32 stays so.
template <typename TO> __device__ __forceinline__ constexpr float most() { return Num<TO>::id == FLAB_FP16 ? 65504.f : 3.38953139e38f; }
template <typename TO> __device__ __forceinline__ TO kept(float z) {
  return Num<TO>::t(fabsf(z) < INFINITY ? fminf(fmaxf(z, -most<TO>()), most<TO>()) : z);
}

struct GemmParams {
  int M, N, K;          // C [M, N]; K: the summed extent
  int tiles_m, tiles_n, tiles;
  int splits, kper;     // the sum in `splits` runs of kper stages; each writes a matrix of its own behind the last one's
  void *c;              // [M, N]
  void *z;              // z before the activation, same type, or null
  const void *bias;     // [N] or null
  const void *res;      // [M, N] or null
  const float *row_scale, *col_scale;  // e4m3 operands
  int act;
  int pairs;            // rows of c, z and res begin on boundaries of two elements
};

template <int BN> struct GemmShape {
  static constexpr int KS = 2;  // blocks of the sum (128 bytes of each row) a stage: one was bound by the stages' hand-over
  static constexpr int S = BN == 64 ? 4 : 3;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BN / 2 * 128, STAGE = KS * (A_BYTES + B_BYTES);
  static constexpr int EPI_WARPS = 8, THREADS = 128 + 32 * EPI_WARPS;
  static constexpr int TURN = BN == 256 ? 4096 : 8192;  // a warp's staging: blocks of 32 rows of 64 bytes, or one of 32 x 32 floats to turn
  static constexpr int BYTES = S * STAGE + EPI_WARPS * TURN + 1024;
};

// TS: outputs by tile stores.  TO: type of c, z, bias, residual.  F8: e4m3 operands, else 16 bits of type T16 (0 fp16, 1 bf16).  AMN / BMN: MN-major operands.
template <typename TO, bool F8, int T16, bool AMN, bool BMN, int BN, bool EPI, bool TS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GemmShape<BN>::THREADS, 1)
    gemm_kernel(const GemmParams p, const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, const __grid_constant__ CUtensorMap mc,
                const __grid_constant__ CUtensorMap mz, const __grid_constant__ CUtensorMap mr) {
  typedef GemmShape<BN> Z;
  constexpr int S = Z::S, KS = Z::KS, BK = F8 ? 128 : 64;  // 128 bytes of each row
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[S], empty[S], acc_full[2], acc_empty[2], res_full[Z::EPI_WARPS][2];
  __shared__ uint32_t tmem_base;
  uint8_t *const buf = raw + ((1024u - (tc::smem_u32(raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_rank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  constexpr uint32_t COLS = 2 * BN;

  if (warp == 2) tc::tmem_alloc_pair(&tmem_base, COLS);
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) tc::mbar_init(&full[i], 1), tc::mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(&acc_full[i], 1), tc::mbar_init(&acc_empty[i], 2 * Z::EPI_WARPS);
    for (int i = 0; i < Z::EPI_WARPS; ++i) tc::mbar_init(&res_full[i][0], 1), tc::mbar_init(&res_full[i][1], 1);
    tc::fence_barrier_init();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
  const int kblocks = (p.K + BK * KS - 1) / (BK * KS), units = p.tiles * p.splits;
  auto run = [&](int unit, int &from, int &to) {  // a unit's blocks of the sum
    from = unit / p.tiles * p.kper;
    to = min(kblocks, from + p.kper);
  };
  auto place = [&](int unit, int &tm, int &tn) {  // groups of 8 rows of tiles, down the group's columns
    const int tile = unit % p.tiles;
    const int group = tile / (8 * p.tiles_n), in = tile - group * 8 * p.tiles_n, high = min(8, p.tiles_m - group * 8);
    tn = in / high;
    tm = group * 8 + in - tn * high;
  };

  // The two loops below are a warp's each: an iteration of theirs is the least that a block of the sum takes, so stages and phases are
  // counted up, and addresses and descriptors added to.
  if (warp == 0) {  // ---- loads
    const bool one = lane == 0;
    if (one) tc::tma_prefetch_desc(&ma), tc::tma_prefetch_desc(&mb);
    const uint32_t bars = tc::peer_addr(&full[0], 0), full0 = tc::smem_u32(&full[0]), empty0 = tc::smem_u32(&empty[0]), stage0 = tc::smem_u32(buf);
    int s = 0;
    uint32_t phase = 1;  // of `empty`: the first round finds every stage free
    bool ok = true;
    for (int unit = cluster; unit < units && ok; unit += clusters) {
      int tm, tn;
      place(unit, tm, tn);
      const int m0 = tm * 256 + rank * 128, n0 = tn * BN + rank * (BN / 2);
      int k0, k1;
      run(unit, k0, k1);
      for (int k = k0 * BK * KS; k < k1 * BK * KS; k += BK * KS) {
        if (!__all_sync(0xffffffffu, tc::mbar_wait(empty0 + s * 8, phase))) {
          tu_tc_error = 730;
          ok = false;
          break;
        }
        const uint32_t bar = bars + s * 8, a = stage0 + s * Z::STAGE, b = a + KS * Z::A_BYTES;
        tc::mbar_expect_tx(one && rank == 0, full0 + s * 8, 2 * Z::STAGE);
#pragma unroll
        for (int h = 0; h < KS; ++h) {  // (a block behind the sum's end arrives as zeros)
          const uint32_t ah = a + h * Z::A_BYTES, bh = b + h * Z::B_BYTES;
          if constexpr (AMN) {
            tc::tma_load_2d_pair(one, ah, &ma, bar, m0, k + h * BK);
            tc::tma_load_2d_pair(one, ah + 8192, &ma, bar, m0 + 64, k + h * BK);
          } else {
            tc::tma_load_2d_pair(one, ah, &ma, bar, k + h * BK, m0);
          }
          if constexpr (BMN) {
#pragma unroll
            for (int i = 0; i < BN / 128; ++i) tc::tma_load_2d_pair(one, bh + i * 8192, &mb, bar, n0 + i * 64, k + h * BK);
          } else {
            tc::tma_load_2d_pair(one, bh, &mb, bar, k + h * BK, n0);
          }
        }
        if (++s == S) s = 0, phase ^= 1;
      }
    }
    __syncwarp();
  } else if (warp == 1) {  // ---- products
    if (rank == 0) {
      constexpr uint32_t idesc = F8 ? tc::instr_desc(256, BN, 0, 0, 0) : tc::instr_desc(256, BN, T16, AMN, BMN);
      // addresses in a descriptor are in 16 bytes; shared memory's stay within its 14 bits
      constexpr uint64_t A_STEP = AMN ? 128 : 2, B_STEP = BMN ? 128 : 2, STAGE_STEP = Z::STAGE / 16;
      const uint32_t at = tc::smem_u32(buf), full0 = tc::smem_u32(&full[0]), empty0 = tc::smem_u32(&empty[0]);
      const uint64_t a0 = AMN ? tc::desc_mnmajor(at, 0, 8192) : tc::desc_kmajor(at, 0, 0);
      const uint64_t b0 = BMN ? tc::desc_mnmajor(at + KS * Z::A_BYTES, 0, 8192) : tc::desc_kmajor(at + KS * Z::A_BYTES, 0, 0);
      const bool one = lane == 0;
      uint64_t ad = a0, bd = b0;
      int s = 0;
      uint32_t phase = 0;
      int n = 0;
      bool ok = true;
      for (int unit = cluster; unit < units && ok; unit += clusters, ++n) {
        const int half = n & 1;
        if (n >= 2 && !__all_sync(0xffffffffu, tc::mbar_wait(&acc_empty[half], (n / 2 - 1) & 1))) {
          tu_tc_error = 731;
          break;
        }
        tc::fence_after_sync();
        const uint32_t d = tmem + half * BN;
        uint32_t add = 0;
        int k0, k1;
        run(unit, k0, k1);
        for (int kb = k1 - k0; kb > 0; --kb) {
          if (!__all_sync(0xffffffffu, tc::mbar_wait(full0 + s * 8, phase))) {
            tu_tc_error = 732;
            ok = false;
            break;
          }
          tc::umma_pair<F8>(one, d, ad, bd, idesc, add);
          add = 1;
#pragma unroll
          for (int k = 1; k < 4 * KS; ++k)
            tc::umma_pair<F8>(one, d, ad + k % 4 * A_STEP + k / 4 * (Z::A_BYTES / 16), bd + k % 4 * B_STEP + k / 4 * (Z::B_BYTES / 16), idesc, 1);
          tc::umma_commit_pair(one, empty0 + s * 8);
          ad += STAGE_STEP, bd += STAGE_STEP;
          if (++s == S) s = 0, phase ^= 1, ad = a0, bd = b0;
        }
        if (ok) tc::umma_commit_pair(one, tc::smem_u32(&acc_full[half]));
      }
    }
    __syncwarp();
  } else if (TS && warp >= 4) {  // ---- epilogue: two warps a quarter of the rows, on blocks of 32 columns in turn
    const int w = warp - 4, quarter = w & 3, side = w >> 2;
    // y and z in turn (y, y, z, z), or where there is room for two blocks only y in turn, or y and z
    uint8_t *const stage = buf + S * Z::STAGE + w * Z::TURN;
    constexpr bool ROOM = Z::TURN == 8192;
    const bool two = ROOM || !EPI || !p.z;
    constexpr int BLOCKS = BN / 64;  // of this warp
    uint32_t seen = 0;  // parity of the residual blocks taken, a bit a buffer
    int n = 0;
    for (int unit = cluster; unit < units; unit += clusters, ++n) {
      const int half = n & 1;
      int tm, tn;
      place(unit, tm, tn);
      const int m0 = tm * 256 + rank * 128 + quarter * 32, n0 = tn * BN + side * 32;
      auto ask = [&](int b) {  // lane 0: the residual of block b, into the buffer that its result will leave from
        const int q = two ? b & 1 : 0;
        tc::mbar_expect_tx(&res_full[w][q], 2048);
        tc::tma_load_2d(stage + q * 2048, &mr, &res_full[w][q], n0 + b * 64, m0);
      };
      if (lane == 0) {
        tc::tma_store_wait_read();
        if (EPI && p.res) ask(0);
      }
      __syncwarp();
      float row_scale = 1.f;
      if (F8 && m0 + lane < p.M) row_scale = p.row_scale[m0 + lane];
      if (!tc::mbar_wait(&acc_full[half], (n / 2) & 1)) {
        tu_tc_error = 733;
        break;
      }
      tc::fence_after_sync();
      const uint32_t from = tmem + half * BN + side * 32 + ((uint32_t)(quarter * 32) << 16);
      bool ok = true;
#pragma unroll 1
      for (int b = 0; b < BLOCKS; ++b) {
        const int q = two ? b & 1 : 0, c = n0 + b * 64;
        float v[32];
        tc::tmem_ld_32x32b_x32(from + b * 64, v);
        if (!two) {
          if (b > 0 && lane == 0) {
            tc::tma_store_wait_read();  // of block b - 1
            if (EPI && p.res && ok) ask(b);
          }
        } else if (EPI && p.res) {
          if (b + 1 < BLOCKS && lane == 0) {
            tc::tma_store_wait_read();  // of block b - 1, a block's work ago
            if (ok) ask(b + 1);  // (behind a wait that ran out nothing is asked for, so that no copy is in flight when the kernel ends)
          }
        } else {
          if (lane == 0) tc::tma_store_wait_read_but_one();  // of block b - 2
        }
        float cs[F8 ? 32 : 1];
        if (F8) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 s = c + 4 * j < p.N ? *reinterpret_cast<const float4 *>(p.col_scale + c + 4 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
            cs[4 * j] = s.x, cs[4 * j + 1] = s.y, cs[4 * j + 2] = s.z, cs[4 * j + 3] = s.w;
          }
        }
        struct alignas(16) Eight {
          TO v[8];
        };
        Eight bias[4];
        if (EPI && p.bias) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + 8 * j < p.N) bias[j] = *reinterpret_cast<const Eight *>(reinterpret_cast<const TO *>(p.bias) + c + 8 * j);
        }
        tc::tmem_ld_wait();
        __syncwarp();
        if (b + 1 == BLOCKS) {  // the warp has taken its last block: the products may use this half again
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_peer(tc::peer_addr(&acc_empty[half], 0));
        }
        if (F8) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = v[j] * row_scale * cs[j];
        }
        if (EPI && p.bias) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += Num<TO>::f(bias[j >> 3].v[j & 7]);
        }
        const int zq = ROOM ? 2 + q : 1;
        // rows of 64 bytes, 64-byte swizzle: 16-byte piece j of row r lies at j ^ (r / 2 % 4)
        auto piece = [&](int buffer, int j) { return reinterpret_cast<Eight *>(stage + buffer * 2048 + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4)); };
        if (EPI && p.z) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            Eight o;
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[8 * j + i])), o.v[i] = Num<TO>::t(v[8 * j + i]);
            if (top > most<TO>()) {  // (asked for eight at a time: held one by one the forward pass took 1 to 2 % longer)
#pragma unroll
              for (int i = 0; i < 8; ++i) o.v[i] = kept<TO>(v[8 * j + i]);
            }
            *piece(zq, j) = o;
          }
        }
        if (EPI && p.act) {
          switch (p.act) {  // one loop an activation, unrolled whole: a loop over v would put it in local memory
            case ACT_SILU:
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = act_fwd(v[j], ACT_SILU);
              break;
            case ACT_SIGMOID:
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = act_fwd(v[j], ACT_SIGMOID);
              break;
            case ACT_LOGSIGMOID:
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = act_fwd(v[j], ACT_LOGSIGMOID);
              break;
            default:
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = act_fwd(v[j], ACT_GELU);
              break;
          }
        }
        if (EPI && p.res) {
          if (ok) {
            ok = tc::mbar_wait(&res_full[w][q], (seen >> q) & 1);
            if (!ok) {
              tu_tc_error = 734;
              if (two && b + 1 < BLOCKS) tc::mbar_wait(&res_full[w][q ^ 1], (seen >> (q ^ 1)) & 1);  // the next block's is on its way
            }
            seen ^= 1u << q;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const Eight r = *piece(q, j);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[8 * j + i] += Num<TO>::f(r.v[i]);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          Eight o;
#pragma unroll
          for (int i = 0; i < 8; ++i) o.v[i] = Num<TO>::t(v[8 * j + i]);
          *piece(q, j) = o;
        }
        tc::fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          tc::tma_store_2d(&mc, stage + q * 2048, c, m0);
          if (EPI && p.z) tc::tma_store_2d(&mz, stage + zq * 2048, c, m0);
          tc::tma_store_commit();
        }
      }
      if (!__all_sync(0xffffffffu, ok)) break;
    }
    if (lane == 0) tc::tma_store_wait_all();
    __syncwarp();
  } else if (!TS && warp >= 4) {  // ---- epilogue: two warps a quarter of the rows, on blocks of 32 columns in turn
    const int w = warp - 4, quarter = w & 3, side = w >> 2;
    float *const turn = reinterpret_cast<float *>(buf + S * Z::STAGE + w * Z::TURN);
    const int odd = lane >> 4, pair = lane & 15;  // this lane's rows 2 i + odd and columns 2 pair, 2 pair + 1 of a block
    struct alignas(2 * sizeof(TO)) Two {
      TO v[2];
    };
    struct Ahead {  // what a block needs from memory
      uint32_t res[16];  // two elements as they lie: nothing waits for a load before the block needs it
      float2 bias, scale;
    };
    int n = 0;
    for (int unit = cluster; unit < units; unit += clusters, ++n) {
      const int half = n & 1;
      int tm, tn;
      place(unit, tm, tn);
      const int m0 = tm * 256 + rank * 128 + quarter * 32, n0 = tn * BN;
      const int rows = min(32, p.M - m0);
      auto ask = [&](int cb, Ahead &a) {
        const int c0 = n0 + cb * 32 + pair * 2;
        const bool on0 = c0 < p.N, on1 = c0 + 1 < p.N;
        a.bias = make_float2(0.f, 0.f), a.scale = make_float2(1.f, 1.f);
        if (EPI && p.bias) {
          if (on0) a.bias.x = Num<TO>::f(reinterpret_cast<const TO *>(p.bias)[c0]);
          if (on1) a.bias.y = Num<TO>::f(reinterpret_cast<const TO *>(p.bias)[c0 + 1]);
        }
        if (F8) {
          if (on0) a.scale.x = p.col_scale[c0];
          if (on1) a.scale.y = p.col_scale[c0 + 1];
        }
        if (EPI && p.res) {
          const unsigned short *e = reinterpret_cast<const unsigned short *>(p.res) + (size_t)(m0 + odd) * p.N + c0;
          if (p.pairs) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (2 * i + odd < rows && on0) a.res[i] = *reinterpret_cast<const uint32_t *>(e + 2 * i * (size_t)p.N);
          } else {
            unsigned short lo[16], hi[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (2 * i + odd < rows && on0) lo[i] = e[2 * i * (size_t)p.N];
              if (2 * i + odd < rows && on1) hi[i] = e[2 * i * (size_t)p.N + 1];
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) a.res[i] = lo[i] | (uint32_t)hi[i] << 16;
          }
        }
      };
      Ahead now, next;
      ask(side, now);
      float row_scale = 0.f;
      if (F8 && lane < rows) row_scale = p.row_scale[m0 + lane];
      if (!tc::mbar_wait(&acc_full[half], (n / 2) & 1)) {
        tu_tc_error = 733;
        break;
      }
      tc::fence_after_sync();
      const uint32_t from = tmem + half * BN + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int cb = side; cb < BN / 32; cb += 2) {
        float v[32];
        tc::tmem_ld_32x32b_x32(from + cb * 32, v);
        tc::tmem_ld_wait();
        if (cb + 2 >= BN / 32) {  // the warp has taken its last block: the products may use this half again
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_peer(tc::peer_addr(&acc_empty[half], 0));
        } else {
          ask(cb + 2, next);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<float4 *>(turn + lane * 32 + ((j ^ (lane & 7)) << 2)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        __syncwarp();
        const int c0 = n0 + cb * 32 + pair * 2;
        const bool on0 = c0 < p.N, on1 = c0 + 1 < p.N;
        float2 f[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = 2 * i + odd;
          f[i] = *reinterpret_cast<const float2 *>(turn + r * 32 + (((pair >> 1) ^ (r & 7)) << 2) + (pair & 1) * 2);
          if (F8) {
            const float rs = __shfl_sync(0xffffffffu, row_scale, r);
            f[i].x = f[i].x * rs * now.scale.x, f[i].y = f[i].y * rs * now.scale.y;
          }
          if (EPI) f[i].x += now.bias.x, f[i].y += now.bias.y;
        }
        auto store = [&](void *q, auto to) {
          TO *e = reinterpret_cast<TO *>(q) + (size_t)(unit / p.tiles) * p.M * p.N + (size_t)(m0 + odd) * p.N + c0;
          if (p.pairs) {
#pragma unroll
            for (int i = 0; i < 16; ++i, e += 2 * (size_t)p.N)
              if (2 * i + odd < rows && on0) {
                Two t;
                t.v[0] = to(f[i].x), t.v[1] = to(f[i].y);
                *reinterpret_cast<Two *>(e) = t;
              }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i, e += 2 * (size_t)p.N) {
              if (2 * i + odd < rows && on0) e[0] = to(f[i].x);
              if (2 * i + odd < rows && on1) e[1] = to(f[i].y);
            }
          }
        };
        if constexpr (EPI) {
          if (p.z) store(p.z, [](float z) { return kept<TO>(z); });
        }
        if (EPI && p.act) {
          switch (p.act) {  // the choice is made once a block
            case ACT_SILU:
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i].x = act_fwd(f[i].x, ACT_SILU), f[i].y = act_fwd(f[i].y, ACT_SILU);
              break;
            case ACT_SIGMOID:
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i].x = act_fwd(f[i].x, ACT_SIGMOID), f[i].y = act_fwd(f[i].y, ACT_SIGMOID);
              break;
            case ACT_LOGSIGMOID:
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i].x = act_fwd(f[i].x, ACT_LOGSIGMOID), f[i].y = act_fwd(f[i].y, ACT_LOGSIGMOID);
              break;
            default:
#pragma unroll
              for (int i = 0; i < 16; ++i) f[i].x = act_fwd(f[i].x, ACT_GELU), f[i].y = act_fwd(f[i].y, ACT_GELU);
              break;
          }
        }
        if constexpr (EPI) {
          if (p.res) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const Two r2 = *reinterpret_cast<const Two *>(&now.res[i]);
              f[i].x += Num<TO>::f(r2.v[0]), f[i].y += Num<TO>::f(r2.v[1]);
            }
          }
        }
        store(p.c, [](float y) { return Num<TO>::t(y); });
        __syncwarp();
        now = next;
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();
  tc::fence_after_sync();
  if (warp == 2) tc::tmem_dealloc_pair(tmem, COLS);
}

// ---- dz = dy act'(z), and the column sums of dz ---------------------------------------------------------------------------
// A block takes 32 V columns x a run of rows; dz may have a row pitch of its own.  Partial column sums, one row a run.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256) act_bwd_kernel(const T *__restrict__ dy, const T *__restrict__ z, T *__restrict__ dz, float *__restrict__ part, int M,
                                                      int N, int pitch, int run) {
  __shared__ float s[8][32 * V];
  struct alignas(V * sizeof(T)) Pack {
    T v[V];
  };
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = (blockIdx.x * 32 + lane) * V;
  const int end = (int)min((long long)M, (blockIdx.y + 1ll) * run);
  auto once = [](const T *at) {  // dy and z are not read again: evict-first loads (79 us without them at 32768 x 2048, 69 with)
    Pack q;
    if constexpr (V == 8) {
      const int4 raw = __ldcs(reinterpret_cast<const int4 *>(at));
      q = *reinterpret_cast<const Pack *>(&raw);
    } else {
      q = *reinterpret_cast<const Pack *>(at);
    }
    return q;
  };
  float sum[V] = {};
  if (c < N) {
#pragma unroll 4
    for (int r = blockIdx.y * run + w; r < end; r += 8) {
      const size_t at = (size_t)r * N + c;
      const Pack d = once(dy + at);
      Pack u, o;
      if (ACT) u = once(z + at);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float f = Num<T>::f(d.v[j]);
        if (ACT) f *= act_slope(Num<T>::f(u.v[j]), ACT);
        sum[j] += f;
        o.v[j] = Num<T>::t(f);
      }
      if (dz) *reinterpret_cast<Pack *>(dz + (size_t)r * pitch + c) = o;
    }
  }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < V; ++j) s[w][lane * V + j] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256)
    if (blockIdx.x * 32 * V + i < N) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) t += s[k][i];
      part[(size_t)blockIdx.y * N + blockIdx.x * 32 * V + i] = t;
    }
}

// Rows of a block, and of a partial column sum: one wave of four blocks an SM over the column groups of `cols` (32768 x 2048: 592
// blocks of 448 rows).
int run_of(int M, int N, int cols) {
  const long long groups = (N + cols - 1) / cols, most = groups < 4ll * sm_count() ? 4ll * sm_count() / groups : 1;
  const long long run = ((M + most - 1) / most + 31) / 32 * 32;
  return (int)run;
}

template <typename T>
int launch_act_bwd(const void *dy, const void *z, void *dz, float *part, int M, int N, int pitch, int act, int &parts, cudaStream_t st) {
  const T *d = reinterpret_cast<const T *>(dy), *u = reinterpret_cast<const T *>(z);
  T *o = reinterpret_cast<T *>(dz);
  bool wide = N % 8 == 0;
  for (const void *q : {(const void *)d, (const void *)u, (const void *)o}) wide = wide && reinterpret_cast<uintptr_t>(q) % 16 == 0;
  const int run = run_of(M, N, wide ? 256 : 32);
  const unsigned runs = (unsigned)((M + (long long)run - 1) / run);
  parts = (int)runs;
  auto launch = [&](auto which) {
    constexpr int ACT = decltype(which)::value;
    if (wide) act_bwd_kernel<T, 8, ACT><<<dim3((N + 255) / 256, runs), 256, 0, st>>>(d, u, o, part, M, N, pitch, run);
    else act_bwd_kernel<T, 1, ACT><<<dim3((N + 31) / 32, runs), 256, 0, st>>>(d, u, o, part, M, N, pitch, run);
    return check_launch("linear_bwd");
  };
  switch (act) {
    case ACT_SILU: return launch(std::integral_constant<int, ACT_SILU>());
    case ACT_SIGMOID: return launch(std::integral_constant<int, ACT_SIGMOID>());
    case ACT_LOGSIGMOID: return launch(std::integral_constant<int, ACT_LOGSIGMOID>());
    case ACT_GELU: return launch(std::integral_constant<int, ACT_GELU>());
    default: return launch(std::integral_constant<int, ACT_NONE>());
  }
}

// Rows of n elements to rows of `pitch`, V elements at a time, for one or two matrices in a launch.
struct Repitch {
  const unsigned short *from;
  unsigned short *to;
  int rows, n, pitch;
};
template <int V> __global__ void __launch_bounds__(256) repitch_kernel(const Repitch a, const Repitch b) {
  struct alignas(2 * V) Pack {
    unsigned short v[V];
  };
  const int lane = threadIdx.x & 31;
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < a.rows + b.rows; r += gridDim.x * 8) {
    const bool second = r >= a.rows;
    const int row = second ? r - a.rows : r, n = second ? b.n : a.n;
    const unsigned short *from = (second ? b.from : a.from) + (size_t)row * n;
    unsigned short *to = (second ? b.to : a.to) + (size_t)row * (second ? b.pitch : a.pitch);
#pragma unroll 8
    for (int c = lane * V; c < n; c += 32 * V) *reinterpret_cast<Pack *>(to + c) = *reinterpret_cast<const Pack *>(from + c);
  }
}

// The joined partial sums of a product in runs, with the epilogue: V elements a thread, the runs in order.
template <typename TO, int V>
__global__ void __launch_bounds__(256) join_kernel(const float *__restrict__ part, int splits, const GemmParams p) {
  struct alignas(sizeof(TO) * V) Out {
    TO v[V];
  };
  struct alignas(V == 1 ? 4 : 8) In {
    float v[V < 2 ? 1 : 2];
  };
  const long long total = (long long)p.M * p.N, at = ((long long)blockIdx.x * 256 + threadIdx.x) * V;
  if (at >= total) return;
  float f[V] = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float *const q = part + s * total + at;
#pragma unroll
    for (int j = 0; j < V; j += sizeof(In) / 4) {
      const In in = *reinterpret_cast<const In *>(q + j);
#pragma unroll
      for (int i = 0; i < (int)(sizeof(In) / 4); ++i) f[j + i] += in.v[i];
    }
  }
  if (p.bias) {
    const int c = (int)(at % p.N);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] += Num<TO>::f(reinterpret_cast<const TO *>(p.bias)[c + j]);
  }
  Out o;
  if (p.z) {
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = kept<TO>(f[j]);
    *reinterpret_cast<Out *>(reinterpret_cast<TO *>(p.z) + at) = o;
  }
  if (p.act) {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = act_fwd(f[j], p.act);
  }
  if (p.res) {
    const Out r = *reinterpret_cast<const Out *>(reinterpret_cast<const TO *>(p.res) + at);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] += Num<TO>::f(r.v[j]);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) o.v[j] = Num<TO>::t(f[j]);
  *reinterpret_cast<Out *>(reinterpret_cast<TO *>(p.c) + at) = o;
}

int operand_map(CUtensorMap *map, const void *base, int dtype, long long rows, int cols, int pitch, int box_cols, int box_rows) {
  const CUtensorMapDataType type = dtype == FLAB_E4M3   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : dtype == FLAB_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, strides[1] = {(uint64_t)pitch * (dtype == FLAB_E4M3 ? 1 : 2)};
  const uint32_t box[2] = {(uint32_t)box_cols, (uint32_t)box_rows};
  const int row = box_cols * (dtype == FLAB_E4M3 ? 1 : 2);  // bytes of a box row: the swizzle's span
  return make_tensor_map(map, base, type, 2, dims, strides, box, row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <typename TO, bool F8, int T16, bool AMN, bool BMN, int BN, bool EPI, bool TS>
int launch_gemm_ts(GemmParams p, const void *a, int a_pitch, const void *b, int b_pitch, int dtype, cudaStream_t st) {
  typedef GemmShape<BN> Z;
  const int bk = F8 ? 128 : 64;
  CUtensorMap ma, mb;
  int rc = AMN ? operand_map(&ma, a, dtype, p.K, p.M, a_pitch, 64, 64) : operand_map(&ma, a, dtype, p.M, p.K, a_pitch, bk, 128);
  if (rc) return rc;
  rc = BMN ? operand_map(&mb, b, dtype, p.K, p.N, b_pitch, 64, 64) : operand_map(&mb, b, dtype, p.N, p.K, b_pitch, bk, BN / 2);
  if (rc) return rc;
  p.tiles_n = (p.N + BN - 1) / BN;
  p.tiles_m = (p.M + 255) / 256;
  const long long tiles = (long long)p.tiles_m * p.tiles_n;
  FLAB_REQUIRE(tiles < (1 << 30), FLAB_E_UNSUPPORTED, "linear: %d x %d is too large", p.M, p.N);
  p.tiles = (int)tiles;
  CUtensorMap mc = ma, mz = ma, mr = ma;  // (a map that is not used may be any)
  if (TS) {
    const int out = Num<TO>::id;
    if ((rc = operand_map(&mc, p.c, out, p.M, p.N, p.N, 32, 32))) return rc;
    if (p.z && (rc = operand_map(&mz, p.z, out, p.M, p.N, p.N, 32, 32))) return rc;
    if (p.res && (rc = operand_map(&mr, p.res, out, p.M, p.N, p.N, 32, 32))) return rc;
  }
  auto kernel = gemm_kernel<TO, F8, T16, AMN, BMN, BN, EPI, TS>;
  if ((rc = set_smem(kernel, Z::BYTES))) return rc;
  const int clusters = sm_count() / 2, units = p.tiles * p.splits;
  kernel<<<2 * (units < clusters ? units : clusters), Z::THREADS, Z::BYTES, st>>>(p, ma, mb, mc, mz, mr);
  return check_launch("linear");
}

template <typename TO, bool F8, int T16, bool AMN, bool BMN, int BN, bool EPI>
int launch_gemm_bn(const GemmParams &p, const void *a, int a_pitch, const void *b, int b_pitch, int dtype, cudaStream_t st) {
  bool ts = sizeof(TO) == 2 && p.N % 8 == 0;
  for (const void *q : {(const void *)p.c, (const void *)p.z, p.res, p.bias, (const void *)p.col_scale}) ts = ts && reinterpret_cast<uintptr_t>(q) % 16 == 0;
  if constexpr (sizeof(TO) == 2) {
    if (ts) return launch_gemm_ts<TO, F8, T16, AMN, BMN, BN, EPI, true>(p, a, a_pitch, b, b_pitch, dtype, st);
  }
  return launch_gemm_ts<TO, F8, T16, AMN, BMN, BN, EPI, false>(p, a, a_pitch, b, b_pitch, dtype, st);
}

// A product's tile width and the number of runs its sum is cut into, by an estimate of its time in us: 4.5 and the rounds of tiles over
// the pairs of SMs times the stages of a run at 0.72, 0.52 and 0.455 us (256, 128 and 64 columns; 4096 x 4096 x 4096: 98, 121 and 210 us, 256 x 2048 x 2048: 16.2, 12.7 and 12.2).  A sum in runs adds the launch that joins
// them (5 us, and 4 for what a second launch costs its caller) and the partial matrices' way through L2.  Cutting pays where few tiles
// have a long sum: 64 x 16384 x 256 60 us in one run, 14.5 in sixteen; 256 x 2048 x 2048 would gain 0.7 of 12.2 us on the device.
struct GemmPlan {
  int bn, splits, kper;
  size_t bytes;  // of partial sums
};
GemmPlan gemm_plan(int M, int N, int K, bool f8, bool bmn) {
  const long long rows = (M + 255ll) / 256, clusters = sm_count() / 2;
  GemmPlan best = {};
  double least = 1e30;
  for (int bn : {256, 128, 64}) {
    if (bmn && bn == 64) continue;
    const int per = f8 ? 256 : 128, kb = (int)((K + (long long)per - 1) / per);  // stages of a sum
    const long long tiles = rows * ((N + bn - 1) / bn);
    for (int want = 1; want <= 64; want *= 2) {
      if (want > 1 && (tiles * want > clusters || kb < 2 * want)) break;
      const int kper = (kb + want - 1) / want, splits = (kb + kper - 1) / kper;
      double us = 4.5 + (double)((tiles * splits + clusters - 1) / clusters) * kper * (bn == 256 ? 0.72 : bn == 128 ? 0.52 : 0.455);
      if (splits > 1) us += 9.0 + 8.0 * splits * M * N / 8.0e6;
      if (us < least) least = us, best = {bn, splits, kper, splits > 1 ? (size_t)splits * M * N * 4 : 0};
    }
  }
  return best;
}

template <typename TO, bool F8, int T16, bool AMN, bool BMN, bool EPI>
int launch_gemm(GemmParams p, const void *a, int a_pitch, const void *b, int b_pitch, int dtype, void *scratch, size_t scratch_bytes, cudaStream_t st) {
  const GemmPlan q = gemm_plan(p.M, p.N, p.K, F8, BMN);
  p.splits = q.splits, p.kper = q.kper;
  auto widths = [&](auto to, auto epi, const GemmParams &g) {
    typedef decltype(to) O;
    constexpr bool E = decltype(epi)::value;
    if (q.bn == 256) return launch_gemm_bn<O, F8, T16, AMN, BMN, 256, E>(g, a, a_pitch, b, b_pitch, dtype, st);
    if constexpr (!BMN) {
      if (q.bn == 64) return launch_gemm_bn<O, F8, T16, AMN, BMN, 64, E>(g, a, a_pitch, b, b_pitch, dtype, st);
    }
    return launch_gemm_bn<O, F8, T16, AMN, BMN, 128, E>(g, a, a_pitch, b, b_pitch, dtype, st);
  };
  if (q.splits == 1) return widths(TO(), std::integral_constant<bool, EPI>(), p);
  FLAB_REQUIRE(scratch && scratch_bytes >= q.bytes && reinterpret_cast<uintptr_t>(scratch) % 256 == 0, FLAB_E_BADARG,
               "linear needs a 256-byte aligned scratch of flab_linear_scratch() or flab_linear_bwd_scratch() bytes");
  GemmParams g = p;
  g.c = scratch, g.z = nullptr, g.bias = g.res = nullptr, g.act = 0, g.pairs = p.N % 2 == 0;
  int rc = widths(float(), std::false_type(), g);
  if (rc) return rc;
  bool wide = p.N % 8 == 0;
  for (const void *r : {(const void *)p.c, (const void *)p.z, p.res}) wide = wide && reinterpret_cast<uintptr_t>(r) % 16 == 0;
  const long long total = (long long)p.M * p.N, per = wide ? 8 : 1;
  const unsigned blocks = (unsigned)((total / per + 255) / 256);
  if (wide) join_kernel<TO, 8><<<blocks, 256, 0, st>>>((const float *)scratch, q.splits, p);
  else join_kernel<TO, 1><<<blocks, 256, 0, st>>>((const float *)scratch, q.splits, p);
  return check_launch("linear join");
}

bool indexed(int M, int N, int K) { return M <= 1 << 30 && N <= 1 << 30 && K <= 1 << 30; }  // by ints, with room for a tile's overhang

template <typename... Ptr> bool four(int n, Ptr... ptr) {
  bool ok = n % 2 == 0;
  for (const void *q : {(const void *)ptr...}) ok = ok && reinterpret_cast<uintptr_t>(q) % 4 == 0;
  return ok;
}

// Operands' rows as TMA needs them (16-byte address and pitch): where they lie, or copied into the caller's scratch.
int pitch_of(int n) { return (n + 7) / 8 * 8; }
bool as_is(const void *p, int n) { return n % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t copy_bytes(long long rows, int n) { return ((size_t)rows * pitch_of(n) * 2 + 255) / 256 * 256; }
struct Operands {
  const void *x, *w;
  size_t bytes;  // of copies in the scratch
};
// x [M, K] and weight [N, K]; with `copied` the scratch holds the copies already (of the forward call)
int operands(Operands &o, const void *x, const void *w, int M, int N, int K, void *ws, size_t ws_bytes, bool copied, cudaStream_t st) {
  o.x = x, o.w = w, o.bytes = 0;
  const size_t xb = as_is(x, K) ? 0 : copy_bytes(M, K), wb = as_is(w, K) ? 0 : copy_bytes(N, K);
  if (xb + wb == 0) return FLAB_OK;
  FLAB_REQUIRE(ws && ws_bytes >= xb + wb, FLAB_E_BADARG, "linear needs a workspace of flab_linear_workspace() bytes");
  char *const at = reinterpret_cast<char *>(ws);
  const Repitch a = {(const unsigned short *)x, (unsigned short *)at, xb ? M : 0, K, pitch_of(K)};
  const Repitch b = {(const unsigned short *)w, (unsigned short *)(at + xb), wb ? N : 0, K, pitch_of(K)};
  o.bytes = xb + wb;
  if (xb) o.x = a.to;
  if (wb) o.w = b.to;
  if (copied) return FLAB_OK;
  const int blocks = (a.rows + b.rows + 7) / 8, cap = sm_count() * 8, grid = blocks < cap ? blocks : cap;
  int by = K % 4 == 0 ? 4 : K % 2 == 0 ? 2 : 1;
  while (by > 1 && ((xb && reinterpret_cast<uintptr_t>(x) % (2 * by)) || (wb && reinterpret_cast<uintptr_t>(w) % (2 * by)))) by /= 2;
  if (by == 4) repitch_kernel<4><<<grid, 256, 0, st>>>(a, b);
  else if (by == 2) repitch_kernel<2><<<grid, 256, 0, st>>>(a, b);
  else repitch_kernel<1><<<grid, 256, 0, st>>>(a, b);
  return check_launch("linear repitch");
}

}  // namespace

int sum_partials(const float *part, void *out, int parts, int n, int dtype, cudaStream_t st);

}  // namespace flab

extern "C" {

size_t flab_linear_workspace(const void *x, const void *weight, int M, int N, int K) {
  using namespace flab;
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return (as_is(x, K) ? 0 : copy_bytes(M, K)) + (as_is(weight, K) ? 0 : copy_bytes(N, K));
}

size_t flab_linear_scratch(int M, int N, int K, int dtype) {
  using namespace flab;
  return M <= 0 || N <= 0 || K <= 0 ? 0 : gemm_plan(M, N, K, dtype == FLAB_E4M3, false).bytes;
}

size_t flab_linear_bwd_scratch(const void *dy, int M, int N, int K, int act) {
  using namespace flab;
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const size_t a = gemm_plan(M, K, N, false, true).bytes, b = gemm_plan(N, K, M, false, true).bytes;
  return (act == ACT_NONE && as_is(dy, N) ? 0 : copy_bytes(M, N)) + (a > b ? a : b);
}

int flab_linear_fwd(const void *x, const void *weight, const void *bias, const void *residual, void *y, void *z, int M, int N, int K, int act, int dtype,
                    void *ws, size_t ws_bytes, void *scratch, size_t scratch_bytes, void *stream) {
  using namespace flab;
  cudaStream_t st = (cudaStream_t)stream;
  FLAB_REQUIRE(M >= 0 && N > 0 && K > 0 && act >= 0 && act <= ACT_GELU, FLAB_E_BADARG, "linear_fwd: M = %d, N = %d, K = %d or activation %d", M, N, K, act);
  FLAB_REQUIRE(indexed(M, N, K), FLAB_E_UNSUPPORTED, "linear_fwd: sides beyond 2^30");
  FLAB_REQUIRE(dtype == FLAB_BF16 || dtype == FLAB_FP16, FLAB_E_UNSUPPORTED, "linear_fwd: element type %d is not supported", dtype);
  if (M == 0) return FLAB_OK;
  FLAB_REQUIRE(x && weight && y, FLAB_E_BADARG, "linear_fwd needs x, weight, y");
  FLAB_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 256 == 0, FLAB_E_BADARG, "linear_fwd: ws must be 256-byte aligned");
  Operands o;
  int rc = operands(o, x, weight, M, N, K, ws, ws_bytes, false, st);
  if (rc) return rc;
  GemmParams p = {};
  p.M = M, p.N = N, p.K = K, p.c = y, p.z = z, p.bias = bias, p.res = residual, p.act = act;
  p.pairs = four(N, y, z, residual);
  const int kp = pitch_of(K);
  return dtype == FLAB_BF16 ? launch_gemm<bf16, false, 1, false, false, true>(p, o.x, kp, o.w, kp, dtype, scratch, scratch_bytes, st)
                            : launch_gemm<__half, false, 0, false, false, true>(p, o.x, kp, o.w, kp, dtype, scratch, scratch_bytes, st);
}

int flab_linear_bwd_partials(int M, int N) {
  if (M <= 0 || N <= 0) return 1;
  long long most = 1;
  for (int cols : {256, 32}) {
    const int run = flab::run_of(M, N, cols);
    const long long runs = (M + (long long)run - 1) / run;
    most = runs > most ? runs : most;
  }
  return (int)most;
}

int flab_linear_bwd(const void *x, const void *weight, const void *z, const void *dy, void *dx, void *dweight, void *dbias, float *db_partial, int M, int N,
                    int K, int act, int dtype, void *ws, size_t ws_bytes, void *scratch, size_t scratch_bytes, void *stream) {
  using namespace flab;
  cudaStream_t st = (cudaStream_t)stream;
  FLAB_REQUIRE(M > 0 && N > 0 && K > 0 && act >= 0 && act <= ACT_GELU, FLAB_E_BADARG, "linear_bwd: M = %d, N = %d, K = %d or activation %d", M, N, K, act);
  FLAB_REQUIRE(indexed(M, N, K), FLAB_E_UNSUPPORTED, "linear_bwd: sides beyond 2^30");
  FLAB_REQUIRE(dtype == FLAB_BF16 || dtype == FLAB_FP16, FLAB_E_UNSUPPORTED, "linear_bwd: element type %d is not supported", dtype);
  FLAB_REQUIRE(dy && ((!dx && !dweight) || (x && weight)) && (act == ACT_NONE || z) && (!dbias || db_partial), FLAB_E_BADARG,
               "linear_bwd needs dy, x and weight for dx or dweight, z for an activation, db_partial for dbias");
  FLAB_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 256 == 0 && reinterpret_cast<uintptr_t>(scratch) % 256 == 0, FLAB_E_BADARG,
               "linear_bwd: ws and scratch must be 256-byte aligned");
  Operands o = {x, weight, 0};
  int rc = dx || dweight ? operands(o, x, weight, M, N, K, ws, ws_bytes, true, st) : FLAB_OK;
  if (rc) return rc;
  const void *dz = dy;
  const int zp = pitch_of(N), kp = pitch_of(K);
  const size_t dz_bytes = act == ACT_NONE && as_is(dy, N) ? 0 : copy_bytes(M, N);
  const bool make_dz = (dx || dweight) && dz_bytes;
  char *part = reinterpret_cast<char *>(scratch);  // of partial sums, behind dz
  size_t part_bytes = scratch_bytes;
  if (make_dz || dbias) {
    void *out = nullptr;
    if (make_dz) {
      FLAB_REQUIRE(scratch && scratch_bytes >= dz_bytes, FLAB_E_BADARG, "linear_bwd needs a scratch of flab_linear_bwd_scratch() bytes");
      dz = out = scratch;
      part += dz_bytes, part_bytes -= dz_bytes;
    }
    int parts = 0;
    rc = dtype == FLAB_BF16 ? launch_act_bwd<bf16>(dy, z, out, dbias ? db_partial : nullptr, M, N, zp, act, parts, st)
                            : launch_act_bwd<__half>(dy, z, out, dbias ? db_partial : nullptr, M, N, zp, act, parts, st);
    if (rc) return rc;
    if (dbias && (rc = sum_partials(db_partial, dbias, parts, N, dtype, st))) return rc;
  }
  GemmParams p = {};
  if (dx) {
    p.M = M, p.N = K, p.K = N, p.c = dx, p.pairs = four(K, dx);
    rc = dtype == FLAB_BF16 ? launch_gemm<bf16, false, 1, false, true, false>(p, dz, zp, o.w, kp, dtype, part, part_bytes, st)
                            : launch_gemm<__half, false, 0, false, true, false>(p, dz, zp, o.w, kp, dtype, part, part_bytes, st);
    if (rc) return rc;
  }
  if (dweight) {
    p.M = N, p.N = K, p.K = M, p.c = dweight, p.pairs = four(K, dweight);
    rc = dtype == FLAB_BF16 ? launch_gemm<bf16, false, 1, true, true, false>(p, dz, zp, o.x, kp, dtype, part, part_bytes, st)
                            : launch_gemm<__half, false, 0, true, true, false>(p, dz, zp, o.x, kp, dtype, part, part_bytes, st);
    if (rc) return rc;
  }
  return FLAB_OK;
}

int flab_linear_e4m3(const void *x, const float *x_scale, const void *weight, const float *w_scale, const void *bias, const void *residual, void *y, int M,
                     int N, int K, int act, int out_dtype, void *scratch, size_t scratch_bytes, void *stream) {
  using namespace flab;
  cudaStream_t st = (cudaStream_t)stream;
  FLAB_REQUIRE(M >= 0 && N > 0 && K > 0 && act >= 0 && act <= ACT_GELU, FLAB_E_BADARG, "linear_e4m3: M = %d, N = %d, K = %d or activation %d", M, N, K, act);
  FLAB_REQUIRE(indexed(M, N, K), FLAB_E_UNSUPPORTED, "linear_e4m3: sides beyond 2^30");
  FLAB_REQUIRE(out_dtype == FLAB_BF16 || out_dtype == FLAB_FP16, FLAB_E_UNSUPPORTED, "linear_e4m3: output type %d is not supported", out_dtype);
  if (M == 0) return FLAB_OK;
  FLAB_REQUIRE(x && x_scale && weight && w_scale && y, FLAB_E_BADARG, "linear_e4m3 needs x, weight, their scales and y");
  FLAB_REQUIRE(K % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(weight) % 16 == 0, FLAB_E_UNSUPPORTED,
               "linear_e4m3: K = %d must be a multiple of 16 and the operands 16-byte aligned", K);
  GemmParams p = {};
  p.M = M, p.N = N, p.K = K, p.c = y, p.bias = bias, p.res = residual, p.act = act, p.row_scale = x_scale, p.col_scale = w_scale;
  p.pairs = four(N, y, residual);
  return out_dtype == FLAB_BF16 ? launch_gemm<bf16, true, 0, false, false, true>(p, x, K, weight, K, FLAB_E4M3, scratch, scratch_bytes, st)
                                : launch_gemm<__half, true, 0, false, false, true>(p, x, K, weight, K, FLAB_E4M3, scratch, scratch_bytes, st);
}
}
