// linear16.cu -- linear layer on 16-bit operands,
//   out = residual + gate o act(x w^T + bias),
// on the 5th-generation tensor cores (kind::f16, FP32 accumulators in TMEM),
// with bias, activation, gate and residual applied to the accumulators, so the
// only traffic is x, w, the residual and the output.
//
// Two kernels, chosen by the number of rows M:
//   * pair kernel (M > kSkinnyRows): CTA pairs, 256 x bn output tiles
//     (x on the M side), persistent, the epilogue of one tile under the main
//     loop of the next.  Bound by the tensor cores.
//   * skinny kernel (M <= kSkinnyRows): the weights on the M side (128 rows of
//     w per CTA), the x rows as the N side, K split over the CTAs of a
//     cluster.  Bound by the bytes of w.
#include "qi_internal.h"
#include "sm100.cuh"

#include <type_traits>

namespace qi {
namespace {

__device__ int g_linear16_err;  // set by a bounded wait that gave up (linear16_take_error)

constexpr int kSkinnyRows = 128;
constexpr int BK = 64;  // K elements per pipeline stage: 128 bytes, one swizzle row

struct alignas(64) L16Dev {
  CUtensorMap tmX, tmW, tmO, tmR;  // x, w; output and residual (pair kernel)
  const void* bias;
  const float* gate;
  const void* residual;
  void* out;
  long long ldr, ldo;
  int M, N, K, act;
  int bn, tiles_m, tiles_n;  // pair kernel
  int tn, stages, splits;    // skinny kernel
};

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float cvt_in(float v) { return v; }
__device__ __forceinline__ float cvt_in(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float cvt_in(__half v) { return __half2float(v); }
template <typename O>
__device__ __forceinline__ O cvt_out(float v);
template <>
__device__ __forceinline__ float cvt_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 cvt_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half cvt_out<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float sigmoid_f32(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }
// 0.5 v (1 + tanh u) = v sigmoid(2u), u = sqrt(2/pi) (v + 0.044715 v^3): the
// exponential keeps full FP32 accuracy where the hardware tanh has 11 bits.
__device__ __forceinline__ float gelu_f32(float v) {
  return v * sigmoid_f32(1.5957691216057308f * (v + 0.044715f * v * v * v));
}
__device__ __forceinline__ float activate(float v, int act) {
  return act == QI_ACT_GELU ? gelu_f32(v) : (act == QI_ACT_SILU ? v * sigmoid_f32(v) : v);
}

template <typename T>
constexpr uint32_t idesc16(int M, int N) {
  return std::is_same<T, __nv_bfloat16>::value ? idesc_bf16(M, N) : idesc_f16(M, N, false, false);
}

// v[0..31] += p[0..n_valid) (a bias slice; the columns past it are clipped).
template <typename T>
__device__ __forceinline__ void add_bias32(float (&v)[32], const T* p, int n_valid) {
  if (n_valid >= 32 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const uint4* p4 = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 w = __ldg(p4 + i);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2<T>(u[e]);
        v[8 * i + 2 * e] += f.x;
        v[8 * i + 2 * e + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < n_valid) v[j] += cvt_in(p[j]);
  }
}

// ------------------------------------------------------------------ pair kernel
namespace pk {
constexpr int BM = 256, BN_MAX = 256;
constexpr int A_BYTES = 128 * BK * 2;         // this CTA's 128 rows of x
constexpr int B_BYTES = BN_MAX / 2 * BK * 2;  // this CTA's half of the tile's w rows
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
// staging sub-tile of one epilogue warp: 32 rows x 32 columns of the output
template <typename O>
constexpr int sub_bytes() { return 32 * 32 * static_cast<int>(sizeof(O)); }
// 2-byte outputs leave room for a sixth stage
template <typename O>
constexpr int stages() { return sizeof(O) == 4 ? 5 : 6; }
template <typename O>
constexpr int smem_bytes() {
  return 1024 + stages<O>() * (A_BYTES + B_BYTES) + EPI_WARPS * 2 * sub_bytes<O>() + 512;
}
}  // namespace pk

// Tile t of the persistent loop: groups of 8 row blocks, rows fastest within a
// group, so that the tiles running at one time share x and w panels in L2.
__device__ __forceinline__ void pair_tile(const L16Dev& a, int t, int& m0, int& n0) {
  const int per = 8 * a.tiles_n, g = t / per, r = t - g * per;
  const int rows = min(8, a.tiles_m - g * 8);
  m0 = (g * 8 + r % rows) * pk::BM;
  n0 = r / rows;  // column tile index
}

template <typename T, typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pk::THREADS, 1)
    linear16_pair_kernel(const __grid_constant__ L16Dev args) {
  using namespace pk;
  constexpr int STAGES = stages<O>(), SUB = sub_bytes<O>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint8_t* sE = sB + STAGES * B_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(sE + EPI_WARPS * 2 * SUB);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* xfull = tempty + 2;  // [EPI_WARPS][2] residual sub-tile loaded
  uint64_t* drain = xfull + 2 * EPI_WARPS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cr = cluster_ctarank();
  const bool leader = cr == 0;
  const int cluster = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  const int bn = args.bn, total = args.tiles_m * args.tiles_n;
  const bool wide = args.act == QI_ACT_SWIGLU;
  const int bn_out = wide ? bn / 2 : bn;
  const int kblocks = (args.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * EPI_WARPS);
    }
    for (int b = 0; b < 2 * EPI_WARPS; ++b) mbar_init(&xfull[b], 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&args.tmX);
    tma_prefetch_desc(&args.tmW);
    tma_prefetch_desc(&args.tmO);
    if (args.residual) tma_prefetch_desc(&args.tmR);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before either signals the other
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (lane == 0) {
      const uint32_t full0 = mapa_shared(&full[0], 0);  // the even CTA's stage barriers
      const uint32_t stage_tx = 2 * (A_BYTES + bn / 2 * BK * 2);  // both CTAs' bytes
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = cluster; t < total && ok; t += nclusters) {
        int m0, nt;
        pair_tile(args, t, m0, nt);
        // SwiGLU: the even CTA brings the tile's gate rows of w, the odd CTA
        // its up rows, so accumulator columns [0, bn/2) are the gate products
        const int wrow = wide ? nt * bn_out + static_cast<int>(cr) * args.N : nt * bn + (bn / 2) * static_cast<int>(cr);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          if (leader) mbar_expect_tx(&full[stage], stage_tx);
          const uint32_t fb = full0 + stage * 8;
          tma_load_2d_pair(sA + stage * A_BYTES, &args.tmX, kb * BK, m0 + 128 * static_cast<int>(cr), fb);
          tma_load_2d_pair(sB + stage * B_BYTES, &args.tmW, kb * BK, wrow, fb);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        *abort_flag = 1;
        atomicCAS(&g_linear16_err, 0, kErrTimeoutProducer);
        // copies already issued complete on the even CTA's barrier: give them
        // time to land before this CTA leaves
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) {
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    if (leader) {
      auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
      };
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t idesc = idesc16<T>(BM, 0) | (static_cast<uint32_t>(bn >> 3) << 17);
      const uint64_t ad0 = umma_desc_sw128(smem_u32(sA), 16, 1024), bd0 = umma_desc_sw128(smem_u32(sB), 16, 1024);
      for (int t = cluster; t < total && ok; t += nclusters, ++local) {
        const int buf = local & 1;
        if (!wait_all(&tempty[buf], ((local >> 1) & 1) ^ 1u)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * BN_MAX;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!wait_all(&full[stage], phase)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t ad = ad0 + static_cast<uint64_t>((stage * A_BYTES) >> 4);
          const uint64_t bd = bd0 + static_cast<uint64_t>((stage * B_BYTES) >> 4);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_f16_ss_pair_elect(d_tmem, ad + 2 * k, bd + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
          mma_commit_pair_elect(&empty[stage], 0x3);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        mma_commit_pair_elect(&tfull[buf], 0x3);
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        atomicCAS(&g_linear16_err, 0, kErrTimeoutMma);
      }
      __syncwarp();
      // every MMA issued above (it writes both CTAs' TMEM) completes before teardown
      mma_commit_pair_elect(drain, 0x1);
      const uint64_t t0 = global_timer_ns();
      while (!mbar_try_wait(drain, 0) && global_timer_ns() - t0 < kWaitLimitNs / 4) {
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    // A warp owns 32 rows (its TMEM lane quarter, thread = row) and every
    // second 32-column chunk of the tile: TMEM -> registers -> bias,
    // activation, gate -> swizzled staging sub-tile (already holding the
    // residual, if any) -> TMA store, which clips rows and columns past the
    // end.  Two staging buffers per warp; the next chunk's residual is loaded
    // into the free one meanwhile.
    const int quarter = warp & 3, ew = warp - 2, half = ew >> 2;
    uint8_t* ebuf = sE + ew * 2 * SUB;
    uint64_t* xb = xfull + ew * 2;
    const uint32_t tempty0 = mapa_shared(&tempty[0], 0);
    const bool resid = args.residual != nullptr;
    const T* bias = static_cast<const T*>(args.bias);
    uint32_t xphase = 0, xpending = 0;
    int local = 0, b = 0;
    bool ok = true;
    for (int t = cluster; t < total && ok; t += nclusters, ++local) {
      int m0, nt;
      pair_tile(args, t, m0, nt);
      const int r0 = m0 + 128 * static_cast<int>(cr) + quarter * 32, n0 = nt * bn_out;
      const int buf = local & 1;
      const int nch = min(bn_out, args.N - n0 + 31) / 32;  // chunks that hold a column of the output
      const bool rows_in = r0 < args.M;
      if (resid && rows_in && half < nch && lane == 0) {
        bulk_wait_read<0>();
        mbar_expect_tx(&xb[b], SUB);
        tma_load_2d(ebuf + b * SUB, &args.tmR, n0 + 32 * half, r0, &xb[b]);
        xpending |= 1u << b;
      }
      bool w = mbar_wait(&tfull[buf], (local >> 1) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, w)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t trow = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * BN_MAX;
      for (int c = half; c < nch && rows_in; c += 2, b ^= 1) {
        const int col = n0 + 32 * c;
        uint8_t* sbuf = ebuf + b * SUB;
        uint32_t acc[32];
        float v[32];
        tmem_ld32(trow + 32 * c, acc);
        if (resid) {
          if (lane == 0 && c + 2 < nch) {
            bulk_wait_read<0>();
            mbar_expect_tx(&xb[b ^ 1], SUB);
            tma_load_2d(ebuf + (b ^ 1) * SUB, &args.tmR, col + 64, r0, &xb[b ^ 1]);
            xpending |= 1u << (b ^ 1);
          }
          w = mbar_wait(&xb[b], (xphase >> b) & 1, abort_flag);
          xphase ^= 1u << b;
          xpending &= ~(1u << b);
          if (!__all_sync(0xffffffffu, w)) ok = false;
        } else {
          // the store issued from this buffer two chunks ago must have read it
          if (lane == 0) bulk_wait_read<1>();
          __syncwarp();
        }
        tmem_ld_wait();
        tmem_reg_fence32(acc);
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(acc[j]);
        if (wide) tmem_ld32(trow + bn_out + 32 * c, acc);
        if (bias) add_bias32(v, bias + col, args.N - col);
        if (wide) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= sigmoid_f32(v[j]);
          float u[32];
          tmem_ld_wait();
          tmem_reg_fence32(acc);
#pragma unroll
          for (int j = 0; j < 32; ++j) u[j] = __uint_as_float(acc[j]);
          if (bias) add_bias32(u, bias + args.N + col, args.N - col);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= u[j];
        } else if (args.act == QI_ACT_GELU) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = gelu_f32(v[j]);
        } else if (args.act == QI_ACT_SILU) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= sigmoid_f32(v[j]);
        }
        if (args.gate) {
          if (args.N - col >= 32) {
            const float4* g4 = reinterpret_cast<const float4*>(args.gate + col);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 g = __ldg(g4 + j);
              v[4 * j] *= g.x;
              v[4 * j + 1] *= g.y;
              v[4 * j + 2] *= g.z;
              v[4 * j + 3] *= g.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < args.N - col) v[j] *= args.gate[col + j];
          }
        }
        // row `lane` of the sub-tile, 16-byte pieces swizzled as the TMA
        // boxes are: 64-byte rows (2-byte outputs) or 128-byte rows (FP32)
        if constexpr (sizeof(O) == 4) {
          float4* srow = reinterpret_cast<float4*>(sbuf + lane * 128);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float4 o = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            if (resid) {
              const float4 x = srow[k ^ (lane & 7)];
              o = make_float4(o.x + x.x, o.y + x.y, o.z + x.z, o.w + x.w);
            }
            srow[k ^ (lane & 7)] = o;
          }
        } else {
          uint4* srow = reinterpret_cast<uint4*>(sbuf + lane * 64);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int at = k ^ ((lane >> 1) & 3);
            if (resid) {
              const uint4 x = srow[at];
              const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<O>(xs[e]);
                v[8 * k + 2 * e] += f.x;
                v[8 * k + 2 * e + 1] += f.y;
              }
            }
            srow[at] = make_uint4(pack2<O>(v[8 * k], v[8 * k + 1]), pack2<O>(v[8 * k + 2], v[8 * k + 3]),
                                  pack2<O>(v[8 * k + 4], v[8 * k + 5]), pack2<O>(v[8 * k + 6], v[8 * k + 7]));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&args.tmO, sbuf, col, r0);
          bulk_commit();
        }
      }
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty0 + buf * 8);
    }
    if (lane == 0) {
      bulk_wait<0>();
      for (int i = 0; i < 2; ++i) {  // an abandoned residual load lands before the CTA exits
        if (!(xpending & (1u << i))) continue;
        const uint64_t t0 = global_timer_ns();
        while (!mbar_try_wait(&xb[i], (xphase >> i) & 1) && global_timer_ns() - t0 < kWaitLimitNs / 4) {
        }
      }
    }
    __syncwarp();
    if (!ok && lane == 0) {
      *abort_flag = 1;
      atomicCAS(&g_linear16_err, 0, kErrTimeoutEpilogue);
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs finished with TMEM and each other's barriers
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------------ skinny kernel
// One CTA: 128 rows of w (for SwiGLU 128 gate and 128 up rows) against all of
// x's rows (padded to tn, the MMA's N), over its share of K.  The accumulator's
// TMEM lanes are output columns, so a warp writes 32 neighbouring columns of a
// row at once.  The CTAs of a cluster hold the partial sums of the K splits:
// each puts them into its shared memory as [row][128], and CTA r adds up rows
// r, r + splits, ... over the cluster (in split order: the sum does not depend
// on timing) and runs the epilogue on them.
namespace sk {
constexpr int W_BYTES = 128 * BK * 2;
constexpr int THREADS = 192;
}  // namespace sk

template <typename T, typename O, bool WIDE>
__global__ void __launch_bounds__(sk::THREADS) linear16_skinny_kernel(const __grid_constant__ L16Dev args) {
  using namespace sk;
  constexpr int NW = WIDE ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tn = args.tn, stages = args.stages, splits = args.splits;
  const int x_bytes = tn * BK * 2, stage_bytes = NW * W_BYTES + x_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + stages * stage_bytes);
  uint64_t* empty = full + stages;
  uint64_t* done = empty + stages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits, n0 = (blockIdx.x / splits) * 128;
  const int kblocks = (args.K + BK - 1) / BK;
  const int kb0 = static_cast<int>(static_cast<long long>(kblocks) * rank / splits);
  const int kb1 = static_cast<int>(static_cast<long long>(kblocks) * (rank + 1) / splits);
  const uint32_t cols = NW * tn < 32 ? 32 : NW * tn;  // TMEM columns: a power of two

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&args.tmX);
    tma_prefetch_desc(&args.tmW);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol_w = l2_policy_evict_first(), pol_x = l2_policy_evict_last();
      int stage = 0, last = -1;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        uint8_t* st = smem + stage * stage_bytes;
        mbar_expect_tx(&full[stage], stage_bytes);
        tma_load_2d_hint(st, &args.tmW, kb * BK, n0, &full[stage], pol_w);
        if (WIDE) tma_load_2d_hint(st + W_BYTES, &args.tmW, kb * BK, args.N + n0, &full[stage], pol_w);
        tma_load_2d_hint(st + NW * W_BYTES, &args.tmX, kb * BK, 0, &full[stage], pol_x);
        last = kb - kb0;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) {
        *abort_flag = 1;
        atomicCAS(&g_linear16_err, 0, kErrTimeoutProducer);
        // copies already issued land before the CTA exits
        for (int i = last < stages ? 0 : last - stages + 1; i <= last; ++i) {
          const uint64_t t0 = global_timer_ns();
          while (!mbar_try_wait(&full[i % stages], (i / stages) & 1) && global_timer_ns() - t0 < kWaitLimitNs / 4) {
          }
        }
      }
    }
  } else if (warp == 1) {
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
    };
    const uint32_t idesc = idesc16<T>(128, 0) | (static_cast<uint32_t>(tn >> 3) << 17);
    const uint64_t d0 = umma_desc_sw128(smem_u32(smem), 16, 1024);
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!wait_all(&full[stage], phase)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t wd = d0 + static_cast<uint64_t>((stage * stage_bytes) >> 4);
      const uint64_t xd = wd + static_cast<uint64_t>((NW * W_BYTES) >> 4);
#pragma unroll
      for (int k = 0; k < BK / 16; ++k) {
        const uint32_t more = kb > kb0 || k > 0 ? 1u : 0u;
        mma_f16_ss_elect(tmem_base, wd + 2 * k, xd + 2 * k, idesc, more);
        if (WIDE)
          mma_f16_ss_elect(tmem_base + tn, wd + (W_BYTES >> 4) + 2 * k, xd + 2 * k, idesc, more);
      }
      mma_commit_elect(&empty[stage]);
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      atomicCAS(&g_linear16_err, 0, kErrTimeoutMma);
    }
    __syncwarp();
    mma_commit_elect(done);  // also before teardown after a failed wait
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(done, 0) && global_timer_ns() - t0 < kWaitLimitNs / 4) {
    }
  }

  // epilogue warps: thread = output column (TMEM lane)
  const int quarter = warp & 3, lcol = quarter * 32 + lane, col = n0 + lcol;
  const uint32_t trow = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
  float bias0 = 0.0f, bias1 = 0.0f, gate = 1.0f;
  const bool in = col < args.N;
  if (warp >= 2 && in) {
    const T* bias = static_cast<const T*>(args.bias);
    if (bias) {
      bias0 = cvt_in(bias[col]);
      if (WIDE) bias1 = cvt_in(bias[args.N + col]);
    }
    if (args.gate) gate = args.gate[col];
  }
  // one output element from its sum(s)
  auto finish = [&](int m, float v, float u) {
    v += bias0;
    if (WIDE)
      v = v * sigmoid_f32(v) * (u + bias1);
    else
      v = activate(v, args.act);
    v *= gate;
    if (args.residual) v += cvt_in(static_cast<const O*>(args.residual)[m * args.ldr + col]);
    static_cast<O*>(args.out)[m * args.ldo + col] = cvt_out<O>(v);
  };
  float* part = reinterpret_cast<float*>(smem);  // [NW][M][128] partial sums, over the consumed stages
  if (warp >= 2) {
    const bool w = mbar_wait(done, 0, abort_flag);
    ok = __all_sync(0xffffffffu, w && !*abort_flag);
    if (!ok && lane == 0) {
      *abort_flag = 1;
      atomicCAS(&g_linear16_err, 0, kErrTimeoutEpilogue);
    }
    tc_fence_after();
    if (ok) {
#pragma unroll 1
      for (int c = 0; c < args.M; c += 16) {
        uint32_t r[16], r2[16];
        tmem_ld16(trow + c, r);
        if (WIDE) tmem_ld16(trow + tn + c, r2);
        tmem_ld_wait();
        tmem_reg_fence16(r);
        if (WIDE) tmem_reg_fence16(r2);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (c + j >= args.M) break;
          if (splits == 1) {
            if (in) finish(c + j, __uint_as_float(r[j]), WIDE ? __uint_as_float(r2[j]) : 0.0f);
          } else {
            part[(c + j) * 128 + lcol] = __uint_as_float(r[j]);
            if (WIDE) part[(args.M + c + j) * 128 + lcol] = __uint_as_float(r2[j]);
          }
        }
      }
    }
  }
  if (splits > 1) {
    __syncthreads();
    cluster_sync();
    if (warp >= 2 && in && ok) {
      uint32_t base[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) base[s] = s < splits ? mapa_shared(part, s) + lcol * 4 : 0u;
#pragma unroll 1
      for (int m = rank; m < args.M; m += splits) {
        float v = 0.0f, u = 0.0f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          if (s >= splits) break;
          v += ld_cluster_f32(base[s] + m * 512);
          if (WIDE) u += ld_cluster_f32(base[s] + (args.M + m) * 512);
        }
        finish(m, v, u);
      }
    }
    __syncwarp();
    cluster_sync();  // nobody leaves while its sums are being read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, cols);
  }
}

// ------------------------------------------------------------------ host
template <typename T>
constexpr CUtensorMapDataType tm_type() {
  return std::is_same<T, float>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

template <typename T>
int encode(CUtensorMap* tm, const void* base, long long rows, long long cols, long long ld, int box_cols, int box_rows,
           CUtensorMapSwizzle sw) {
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * sizeof(T)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = qi_encode_tiled(tm, tm_type<T>(), 2, const_cast<void*>(base), dims, strides, box, estr,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? QI_OK : QI_ERR_CUDA;
}

// Pair-tile width: the one whose waves over the SM pairs, times the tile's
// time, finish first.
int pair_width(int M, int cols, bool wide, int clusters) {
  int best = 256;
  double best_t = 1e300;
  for (int bn = 256; bn >= 64; bn -= wide ? 64 : 32) {
    const long long tiles = static_cast<long long>((M + 255) / 256) * ((cols + bn - 1) / bn);
    const double t = static_cast<double>((tiles + clusters - 1) / clusters) * (bn + 48);
    if (t < best_t * 0.97) {
      best = bn;
      best_t = t;
    }
  }
  return best;
}

template <typename T, typename O>
int launch_pair16(const Linear16Args& a, L16Dev& d, cudaStream_t stream, int num_sms) {
  const bool wide = a.act == QI_ACT_SWIGLU;
  const int clusters = num_sms / 2;
  d.bn = pair_width(a.M, (wide ? 2 : 1) * a.N, wide, clusters);
  const int bn_out = wide ? d.bn / 2 : d.bn;
  d.tiles_m = (a.M + pk::BM - 1) / pk::BM;
  d.tiles_n = (a.N + bn_out - 1) / bn_out;
  if (static_cast<long long>(d.tiles_m) * d.tiles_n > 0x7fffffff) return QI_ERR_UNSUPPORTED;
  const CUtensorMapSwizzle osw = sizeof(O) == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (encode<T>(&d.tmX, a.x, a.M, a.K, a.ldx, BK, 128, CU_TENSOR_MAP_SWIZZLE_128B) != QI_OK ||
      encode<T>(&d.tmW, a.w, (wide ? 2ll : 1ll) * a.N, a.K, a.ldw, BK, d.bn / 2, CU_TENSOR_MAP_SWIZZLE_128B) != QI_OK ||
      encode<O>(&d.tmO, a.out, a.M, a.N, a.ldo, 32, 32, osw) != QI_OK ||
      (a.residual && encode<O>(&d.tmR, a.residual, a.M, a.N, a.ldr, 32, 32, osw) != QI_OK))
    return QI_ERR_CUDA;
  static unsigned long long attr_done = 0;
  const auto fn = linear16_pair_kernel<T, O>;
  if (smem_optin(reinterpret_cast<const void*>(fn), pk::smem_bytes<O>(), &attr_done) != QI_OK) return QI_ERR_CUDA;
  const int tiles = d.tiles_m * d.tiles_n;
  fn<<<2 * (tiles < clusters ? tiles : clusters), pk::THREADS, pk::smem_bytes<O>(), stream>>>(d);
  return cudaGetLastError() == cudaSuccess ? QI_OK : QI_ERR_CUDA;
}

template <typename T, typename O, bool WIDE>
int launch_skinny(const Linear16Args& a, L16Dev& d, cudaStream_t stream, int num_sms) {
  constexpr int NW = WIDE ? 2 : 1;
  d.tn = a.M <= 16 ? 16 : (a.M <= 32 ? 32 : (a.M <= 64 ? 64 : 128));
  const int tiles = (a.N + 127) / 128, kblocks = (a.K + BK - 1) / BK;
  // K splits: about one CTA per SM, at least four K blocks each
  int splits = (num_sms - 8 + tiles - 1) / tiles;
  if (splits > kblocks / 4) splits = kblocks / 4;
  d.splits = splits < 1 ? 1 : (splits > 8 ? 8 : splits);
  // stages: two CTAs per SM where three or more of them fit, else one
  const int stage = NW * sk::W_BYTES + d.tn * BK * 2;
  d.stages = (110 * 1024) / stage;
  if (d.stages < 3) d.stages = (220 * 1024) / stage;
  if (d.stages > 8) d.stages = 8;
  const int smem = 1024 + d.stages * stage + 256;
  if (encode<T>(&d.tmX, a.x, a.M, a.K, a.ldx, BK, d.tn, CU_TENSOR_MAP_SWIZZLE_128B) != QI_OK ||
      encode<T>(&d.tmW, a.w, static_cast<long long>(NW) * a.N, a.K, a.ldw, BK, 128, CU_TENSOR_MAP_SWIZZLE_128B) != QI_OK)
    return QI_ERR_CUDA;
  static unsigned long long attr_done = 0;
  const auto fn = linear16_skinny_kernel<T, O, WIDE>;
  if (smem_optin(reinterpret_cast<const void*>(fn), 222 * 1024, &attr_done) != QI_OK) return QI_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles) * d.splits);
  cfg.blockDim = dim3(sk::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = d.splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, static_cast<const L16Dev&>(d)) == cudaSuccess ? QI_OK : QI_ERR_CUDA;
}

template <typename T, typename O>
int launch_typed(const Linear16Args& a, cudaStream_t stream) {
  L16Dev d;
  memset(&d, 0, sizeof(d));
  d.bias = a.bias;
  d.gate = a.gate;
  d.residual = a.residual;
  d.out = a.out;
  d.ldr = a.ldr;
  d.ldo = a.ldo;
  d.M = a.M;
  d.N = a.N;
  d.K = a.K;
  d.act = a.act;
  const int num_sms = device_num_sms();
  if (a.M > kSkinnyRows) return launch_pair16<T, O>(a, d, stream, num_sms);
  return a.act == QI_ACT_SWIGLU ? launch_skinny<T, O, true>(a, d, stream, num_sms)
                                : launch_skinny<T, O, false>(a, d, stream, num_sms);
}

}  // namespace

int linear16_launch(const Linear16Args& a, cudaStream_t stream) {
  if (a.dtype == QI_DT_BF16)
    return a.out_dtype == QI_DT_F32 ? launch_typed<__nv_bfloat16, float>(a, stream)
                                    : launch_typed<__nv_bfloat16, __nv_bfloat16>(a, stream);
  return a.out_dtype == QI_DT_F32 ? launch_typed<__half, float>(a, stream) : launch_typed<__half, __half>(a, stream);
}

int linear16_take_error(int* bad) {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, g_linear16_err, sizeof(int)) != cudaSuccess) return QI_ERR_CUDA;
  if (h) {
    *bad = 1;
    h = 0;
    if (cudaMemcpyToSymbol(g_linear16_err, &h, sizeof(int)) != cudaSuccess) return QI_ERR_CUDA;
  }
  return QI_OK;
}

}  // namespace qi
