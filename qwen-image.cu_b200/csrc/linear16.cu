// linear16.cu -- linear layer on 16-bit operands,
//   out = residual + gate o act(x w^T + bias),
// on the 5th-generation tensor cores (kind::f16, FP32 accumulators in TMEM),
// with bias, activation, gate and residual applied to the accumulators, so the
// only traffic is x, w, the residual and the output.
//
// Two kernels, chosen by the number of rows M of x:
//   * pair kernel: tcgen05 on CTA pairs, 256 x bn output tiles, persistent, the
//     epilogue of one tile under the main loop of the next.  Bound by the tensor
//     cores: 8192 x 12288 x 3584 with GELU 474-496 us (1460-1520 TFLOP/s, tensor
//     cores busy for 97% of the time), back to back under the power cap 575-591.
//     With one wave of narrow tiles by the copies of x and w, about 0.25 us per 64
//     of K.
//   * rows kernel (up to 16 rows): w streamed through warp-level MMAs.  Bound by
//     the bytes of w.
#include "qi_internal.h"
#include "sm100.cuh"

#include <type_traits>

namespace qi {
namespace {

__device__ int g_linear16_err;  // set by a bounded wait that gave up (linear16_take_error)

constexpr int BK = 64;  // K elements per pipeline stage: 128 bytes, one swizzle row

struct alignas(64) L16Dev {  // pair kernel
  CUtensorMap tmX, tmW, tmO, tmR;  // x, w, output, residual
  const void* bias;
  const float* gate;
  const void* residual;  // NULL: none (read through tmR)
  int M, N, K, act;
  int stages, atoms;  // TMA pipeline depth, K blocks per stage
  int bn, tiles_m, tiles_n;
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

// Off by the exponential's documented 2 + floor(1.173 |v|) ulp: 2^-19 up to |v| =
// 12, and more only where it makes up less than 1e-5 of the value or of v.  0 below
// v = -87.3, where the sigmoid is subnormal.
__device__ __forceinline__ float sigmoid_f32(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }
// 0.5 v (1 + tanh u) = v sigmoid(2u), u = sqrt(2/pi) (v + 0.044715 v^3): the
// hardware tanh has 11 bits.
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
      const uint4 w = p4[i];
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
constexpr int A_BLOCK = 128 * BK * 2;  // this CTA's 128 rows of x, one K block
constexpr int MMA_WARP = 2, EPI_WARP0 = 4, EPI_WARPS = 8;  // warps 0 and 1 produce, 3 has no part
constexpr int THREADS = 32 * (EPI_WARP0 + EPI_WARPS);
// sums in parts: registers per thread at launch, then of the first warpgroup and
// of the epilogue's two
constexpr int LAUNCH_REGS = 168, PRODUCER_REGS = 88, EPI_REGS = 208;
static_assert(32 * (EPI_WARP0 * PRODUCER_REGS + EPI_WARPS * EPI_REGS) <= THREADS * LAUNCH_REGS,
              "register split exceeds the launch");
// Sums in parts.  The tensor cores truncate every addition to an accumulator, so
// its error grows with K: 9e-10 K (BF16) or 1.3e-9 K (FP16) of the product in norm,
// with one sign 1.6e-9 or 5e-9 K at small K, 6.7e-9 K (FP16) at large.  Where that
// would show, the epilogue warps take the accumulator over every 768 (BF16) or 512
// (FP16) of K and add it, rounding to nearest, to sums in their registers (128 per
// thread for a 256 x 256 tile); the last part's total goes back to TMEM, where the
// epilogue finds it.  SwiGLU, whose two factors lose in the same direction, takes
// half of that.  Norm error 8e-7 at most for every K, and no warp waits for more of
// K than a part at once.  A part costs 0.24 us, the first MMA on the other
// accumulator (M 8192, N = K = 3584: 148 us as one sum, error 3.9e-6; 156 with
// parts of 768, 163 of 512; SwiGLU, M 1111, N 14336: 172 as one sum, 201).
// It shows in FP32 outputs from one part on; in 16-bit outputs where it reaches a
// quarter of the half step that they are rounded by, with one sign at K = 16384
// (FP16) or 131072 (BF16).
template <typename T>
constexpr int sums_step(bool wide) {  // K blocks, even
  return (std::is_same<T, __half>::value ? 512 : 768) / (wide ? 2 : 1) / BK;
}
template <typename T, typename O>
constexpr int sums_min_k(bool wide) {
  return std::is_same<O, float>::value ? BK * sums_step<T>(wide) : (std::is_same<O, __half>::value ? 16384 : 131072);
}
// staging sub-tile of one epilogue warp: 32 rows x 32 columns of the output
template <typename O>
constexpr int sub_bytes() { return 32 * 32 * static_cast<int>(sizeof(O)); }
constexpr int MAX_STAGES = 8;
constexpr int SMEM_BYTES = 227 * 1024;
// what the stages may take: narrow tiles get more of them
template <typename O>
constexpr int stage_room() { return SMEM_BYTES - 1024 - 512 - EPI_WARPS * 2 * sub_bytes<O>(); }
}  // namespace pk

// Tile t of the persistent loop: groups of 8 row blocks, rows fastest within a
// group, so that the tiles running at one time share x and w panels in L2.
__device__ __forceinline__ void pair_tile(const L16Dev& a, int t, int& m0, int& n0) {
  const int per = 8 * a.tiles_n, g = t / per, r = t - g * per;
  const int rows = min(8, a.tiles_m - g * 8);
  m0 = (g * 8 + r % rows) * pk::BM;
  n0 = r / rows;  // column tile index
}

template <typename T, typename O, bool SUMS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pk::THREADS, 1)
    linear16_pair_kernel(const __grid_constant__ L16Dev args) {
  using namespace pk;
  constexpr int SUB = sub_bytes<O>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stages = args.stages, atoms = args.atoms;
  const int b_block = args.bn / 2 * BK * 2;  // this CTA's half of the tile's w rows, one K block
  const int a_bytes = atoms * A_BLOCK, b_bytes = atoms * b_block;
  uint8_t* sA = smem;
  uint8_t* sB = smem + stages * a_bytes;
  uint8_t* sE = sB + stages * b_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sE + EPI_WARPS * 2 * SUB);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* tfull = empty + MAX_STAGES;
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
  const int kstep = SUMS ? sums_step<T>(wide) : kblocks;  // K blocks per accumulator

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
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
  if (warp == MMA_WARP) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before either signals the other
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_dependency_wait();
  launch_dependents();

  if (warp < EPI_WARP0) {
    if constexpr (SUMS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PRODUCER_REGS));
    if (warp < MMA_WARP) {
      // ------------------------------------------------------------ producers (both CTAs)
      // Warp 0 brings x, warp 1 brings w: waiting for a stage and issuing both
      // copies takes one thread ~430 clocks, more than a narrow tile's MMAs.
      if (lane == 0) {
        const uint32_t full0 = mapa_shared(&full[0], 0);  // the even CTA's stage barriers
        const uint32_t stage_tx = 2 * (a_bytes + b_bytes);  // both CTAs' bytes
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = cluster; t < total && ok; t += nclusters) {
          int m0, nt;
          pair_tile(args, t, m0, nt);
          // SwiGLU: the even CTA brings the tile's gate rows of w, the odd CTA
          // its up rows, so accumulator columns [0, bn/2) are the gate products
          const int wrow = wide ? nt * bn_out + static_cast<int>(cr) * args.N : nt * bn + (bn / 2) * static_cast<int>(cr);
          const int row = warp == 0 ? m0 + 128 * static_cast<int>(cr) : wrow;
          const CUtensorMap* tm = warp == 0 ? &args.tmX : &args.tmW;
          uint8_t* dst = warp == 0 ? sA : sB;
          const int block = warp == 0 ? A_BLOCK : b_block;
          for (int kb = 0; kb < kblocks; kb += atoms) {
            if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag)) {
              ok = false;
              break;
            }
            if (leader && warp == 0) mbar_expect_tx(&full[stage], stage_tx);
            uint8_t* to = dst + stage * atoms * block;
            tma_load_2d_pair(to, tm, kb * BK, row, full0 + stage * 8);
            if (atoms == 2) tma_load_2d_pair(to + block, tm, (kb + 1) * BK, row, full0 + stage * 8);  // past K: zeros
            if (++stage == stages) {
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
    } else if (warp == MMA_WARP) {
      // ------------------------------------------------------------ MMA issuer (even CTA)
      if (leader) {
        auto wait_all = [&](uint64_t* bar, uint32_t parity) {
          return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
        };
        int stage = 0, local = 0;
        uint32_t phase = 0;
        bool ok = true, ready = mbar_test_wait(&full[0], 0);
        const uint32_t idesc = idesc16<T>(BM, 0) | (static_cast<uint32_t>(bn >> 3) << 17);
        const uint64_t ad0 = umma_desc_sw128(smem_u32(sA), 16, 1024), bd0 = umma_desc_sw128(smem_u32(sB), 16, 1024);
        for (int t = cluster; t < total && ok; t += nclusters) {
          for (int k0 = 0; k0 < kblocks && ok; k0 += kstep, ++local) {
            const int buf = local & 1, k1 = min(kblocks, k0 + kstep);
            if (!wait_all(&tempty[buf], ((local >> 1) & 1) ^ 1u)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + buf * BN_MAX;
            for (int kb = k0; kb < k1; kb += atoms) {
              if (!__all_sync(0xffffffffu, ready) && !wait_all(&full[stage], phase)) {
                ok = false;
                break;
              }
              tc_fence_after();
              const int cur = stage;
              if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
              }
              ready = mbar_test_wait(&full[stage], phase);
              uint64_t ad = ad0 + static_cast<uint64_t>((cur * a_bytes) >> 4);
              uint64_t bd = bd0 + static_cast<uint64_t>((cur * b_bytes) >> 4);
#pragma unroll
              for (int k = 0; k < BK / 16; ++k)
                mma_f16_ss_pair_elect(d_tmem, ad + 2 * k, bd + 2 * k, idesc, kb > k0 || k > 0 ? 1u : 0u);
              if (atoms == 2) {
                ad += A_BLOCK >> 4;
                bd += static_cast<uint64_t>(b_block >> 4);
#pragma unroll
                for (int k = 0; k < BK / 16; ++k) mma_f16_ss_pair_elect(d_tmem, ad + 2 * k, bd + 2 * k, idesc, 1u);
              }
              mma_commit_pair_elect(&empty[cur], 0x3);
            }
            if (!ok) break;
            mma_commit_pair_elect(&tfull[buf], 0x3);
          }
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
    }
  } else {
    if constexpr (SUMS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(EPI_REGS));
    // ------------------------------------------------------------ epilogue (both CTAs)
    // A warp owns 32 rows (its TMEM lane quarter, thread = row) and every
    // second 32-column chunk of the tile: TMEM -> registers -> bias,
    // activation, gate -> swizzled staging sub-tile (already holding the
    // residual, if any) -> TMA store, which clips rows and columns past the
    // end.  Two staging buffers per warp; the next chunk's residual is loaded
    // into the free one meanwhile.
    const int quarter = warp & 3, ew = warp - EPI_WARP0, half = ew >> 2;
    uint8_t* ebuf = sE + ew * 2 * SUB;
    uint64_t* xb = xfull + ew * 2;
    const uint32_t tempty0 = mapa_shared(&tempty[0], 0);
    const bool resid = args.residual != nullptr;
    const T* bias = static_cast<const T*>(args.bias);
    uint32_t xphase = 0, xpending = 0;
    int local = 0, b = 0;
    bool ok = true;
    for (int t = cluster; t < total && ok; t += nclusters) {
      int m0, nt;
      pair_tile(args, t, m0, nt);
      const int r0 = m0 + 128 * static_cast<int>(cr) + quarter * 32, n0 = nt * bn_out;
      const int nch = min(bn_out, args.N - n0 + 31) / 32;  // chunks that hold a column of the output
      const bool rows_in = r0 < args.M;
      if (resid && rows_in && half < nch && lane == 0) {
        bulk_wait_read<0>();
        mbar_expect_tx(&xb[b], SUB);
        tma_load_2d(ebuf + b * SUB, &args.tmR, n0 + 32 * half, r0, &xb[b]);
        xpending |= 1u << b;
      }
      const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      bool w = true;
      int buf = local & 1;
      if constexpr (SUMS) {
        // this warp's chunks, four at most (SwiGLU: two of gate, two of up)
        float sum[4][32] = {};
        auto at = [&](int i) { return lanes + buf * BN_MAX + 32 * half + (wide ? 64 * (i & 1) + (i >> 1) * bn_out : 64 * i); };
        const int mine = rows_in ? (nch - half + 1) / 2 : 0;
        auto has = [&](int i) { return (wide ? i & 1 : i) < mine; };
        for (int k0 = 0;; ++local) {
          buf = local & 1;
          w = mbar_wait(&tfull[buf], (local >> 1) & 1, abort_flag);
          if (!__all_sync(0xffffffffu, w)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (has(i)) {
              uint32_t acc[32];
              tmem_ld32(at(i), acc);
              tmem_ld_wait();
              tmem_reg_fence32(acc);
#pragma unroll
              for (int j = 0; j < 32; ++j) sum[i][j] += __uint_as_float(acc[j]);
            }
          k0 += kstep;
          if (k0 >= kblocks) break;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(tempty0 + buf * 8);
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (has(i)) tmem_st32(at(i), *reinterpret_cast<uint32_t(*)[32]>(sum[i]));
        tmem_st_wait();
      } else {
        w = mbar_wait(&tfull[buf], (local >> 1) & 1, abort_flag);
        if (!__all_sync(0xffffffffu, w)) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
      const uint32_t trow = lanes + buf * BN_MAX;
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
              const float4 g = g4[j];
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
      ++local;
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
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------------ rows kernel
// Few rows of x: the bytes of w are what counts, so w goes from HBM straight to
// the registers of warp-level MMAs (m16n8k16: 16 rows of w, 8 rows of x), every
// load 16 bytes per thread and several in flight, with no staging to wait for.
// The K index of an MMA is a summation index, so its order is free: a thread's
// 16 bytes (8 neighbouring k) are taken as its slots of two MMAs, for w and x
// alike.  A CTA makes 16 columns (SwiGLU: 16 gate and 16 up rows of w); its 8
// warps take 32-k blocks of K in turn and add up in shared memory, in warp
// order.  One row, N = K = 3584 (25.7 MB of w): 9.8 us; a kernel that only reads
// those bytes takes 8.1-8.7 us from launch to launch.
namespace rk {
constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int UNROLL = 4;  // 32-k blocks whose loads are in flight per warp
// Steps of the K loop after which a warp adds its accumulators, rounding to
// nearest, to its sums in shared memory: 512 of its K, 4096 of the whole, SwiGLU
// half (see Sums in parts above).
constexpr int sums_steps(bool wide) { return (wide ? 256 : 512) / (32 * UNROLL); }
}  // namespace rk

template <typename T>
__device__ __forceinline__ void mma_m16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  if (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight neighbouring k of a row from k on, zeros from K on.
template <typename T, bool STREAM>
__device__ __forceinline__ uint4 load8(const T* row, int k, int K) {
  if (k + 8 <= K) {
    uint4 v;
    if (STREAM)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                   : "l"(row + k));
    else
      v = *reinterpret_cast<const uint4*>(row + k);
    return v;
  }
  uint32_t u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (k + e < K) u[e >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[k + e]) << (16 * (e & 1));
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// G: groups of 8 rows of x; R: 16-row tiles of w per warp (SwiGLU: gate, up).
template <typename T, typename O, int G, int R, bool WIDE>
__global__ void __launch_bounds__(rk::THREADS) linear16_rows_kernel(const __grid_constant__ Linear16Args args) {
  using namespace rk;
  constexpr int COLS = WIDE ? 16 : 16 * R;               // output columns of the CTA
  constexpr int STRIDE = 16 * R + 4;                     // floats per x row in shared memory: conflict-free stores
  constexpr int SWEEPS = (8 * G * COLS + THREADS - 1) / THREADS;
  extern __shared__ float red[];                         // [WARPS][8 G][STRIDE]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * COLS;
  const long long last = (WIDE ? 2ll : 1ll) * args.N - 1;
  const T* wrow[R][2];  // rows g and g + 8 of each tile; past the end the last row, whose sums nobody reads
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      long long n = n0 + g + 8 * h + (WIDE ? static_cast<long long>(r) * args.N : 16 * r);
      if (n > last) n = last;
      wrow[r][h] = static_cast<const T*>(args.w) + n * args.ldw;
    }
  const T* xrow[G];
#pragma unroll
  for (int j = 0; j < G; ++j) xrow[j] = static_cast<const T*>(args.x) + min(8 * j + g, args.M - 1) * args.ldx;
  grid_dependency_wait();
  launch_dependents();

  // this thread's outputs: column n0 + c, rows m0, m0 + THREADS / COLS, ...
  const int c = threadIdx.x % COLS, m0 = threadIdx.x / COLS, col = n0 + c;
  const bool in = col < args.N;
  float bias0 = 0.0f, bias1 = 0.0f, gate = 1.0f;
  O res[SWEEPS];
  if (in) {
    const T* bias = static_cast<const T*>(args.bias);
    if (bias) bias0 = cvt_in(bias[col]);
    if (WIDE && bias) bias1 = cvt_in(bias[args.N + col]);
    if (args.gate) gate = args.gate[col];
    if (args.residual) {
#pragma unroll
      for (int i = 0; i < SWEEPS; ++i) {
        const long long m = m0 + i * (THREADS / COLS);
        if (m < args.M) res[i] = static_cast<const O*>(args.residual)[m * args.ldr + col];
      }
    }
  }

  float acc[R][G][4] = {};
  const int kblocks = (args.K + 31) / 32;
  // this thread's sums: its accumulators, added to what it had put there before
  bool summed = false;
  auto put = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < G; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float* p = red + (warp * 8 * G + 8 * j + 2 * t + (e & 1)) * STRIDE + 16 * r + g + 8 * (e >> 1);
          *p = summed ? *p + acc[r][j][e] : acc[r][j][e];
          acc[r][j][e] = 0.0f;
        }
    summed = true;
  };
  int steps = 0;
#pragma unroll 1
  for (int kb = warp; kb < kblocks; kb += WARPS * UNROLL) {
    uint4 w[UNROLL][R][2];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int k = (kb + u * WARPS) * 32 + 8 * t;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        w[u][r][0] = load8<T, true>(wrow[r][0], k, args.K);
        w[u][r][1] = load8<T, true>(wrow[r][1], k, args.K);
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int k = (kb + u * WARPS) * 32 + 8 * t;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const uint4 x = load8<T, false>(xrow[j], k, args.K);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          mma_m16n8k16<T>(acc[r][j], w[u][r][0].x, w[u][r][1].x, w[u][r][0].y, w[u][r][1].y, x.x, x.y);
          mma_m16n8k16<T>(acc[r][j], w[u][r][0].z, w[u][r][1].z, w[u][r][0].w, w[u][r][1].w, x.z, x.w);
        }
      }
    }
    if (++steps == sums_steps(WIDE)) {
      steps = 0;
      put();
    }
  }
  put();
  __syncthreads();
  if (!in) return;
#pragma unroll
  for (int i = 0; i < SWEEPS; ++i) {
    const int m = m0 + i * (THREADS / COLS);
    if (m >= args.M) break;
    float v = 0.0f, u = 0.0f;
#pragma unroll
    for (int q = 0; q < WARPS; ++q) {
      const float* p = red + (q * 8 * G + m) * STRIDE + c;
      v += p[0];
      if (WIDE) u += p[16];
    }
    v += bias0;
    if (WIDE)
      v = v * sigmoid_f32(v) * (u + bias1);
    else
      v = activate(v, args.act);
    v *= gate;
    if (args.residual) v += cvt_in(res[i]);
    static_cast<O*>(args.out)[m * args.ldo + col] = cvt_out<O>(v);
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

// An operand [rows, K], K tail filled with zeros: boxes of one atom.
template <typename T>
int encode_operand(CUtensorMap* tm, const void* base, long long rows, int K, long long ld, int box_rows) {
  return encode<T>(tm, base, rows, K, ld, BK, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Pair-tile width: the one whose waves over the SM pairs, times the tile's
// time, finish first.  The 48 stand for what a K block costs at any width (1024
// rows x 4608 x 3584: 256 wide, one wave, 25.4 us; 128 wide, two, 29.2 us).
int pair_width(int M, int cols, bool wide, int clusters) {
  int best = pk::BN_MAX;
  double best_t = 1e300;
  for (int bn = pk::BN_MAX; bn >= 64; bn -= wide ? 64 : 32) {
    const long long tiles = static_cast<long long>((M + 255) / 256) * ((cols + bn - 1) / bn);
    const double t = static_cast<double>((tiles + clusters - 1) / clusters) * (bn + 48);
    if (t < best_t * 0.97) {
      best = bn;
      best_t = t;
    }
  }
  return best;
}

// Launch with the dependent-launch attribute (see grid_dependency_wait).
template <typename A>
int launch16(void (*fn)(const A), unsigned grid, int threads, int smem, const A& args, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, fn, args) == cudaSuccess) return QI_OK;
  cudaGetLastError();  // reported by status, not left for the caller's next check
  return QI_ERR_CUDA;
}

template <typename T, typename O, bool SUMS>
int launch_pair16(const Linear16Args& a, L16Dev& d, cudaStream_t stream, int num_sms) {
  const bool wide = a.act == QI_ACT_SWIGLU;
  const int clusters = num_sms / 2;
  d.bn = pair_width(a.M, (wide ? 2 : 1) * a.N, wide, clusters);
  const int bn_out = wide ? d.bn / 2 : d.bn;
  d.tiles_m = (a.M + pk::BM - 1) / pk::BM;
  d.tiles_n = (a.N + bn_out - 1) / bn_out;
  if (static_cast<long long>(d.tiles_m) * d.tiles_n > 0x3fffffff) return QI_ERR_UNSUPPORTED;
  // Two K blocks per stage for narrow tiles, where a stage's waits and barriers
  // cost more than one block of MMAs (N 4608, K 3584, one / two: 96 rows 17.5 /
  // 15.7 us, 512 rows 18.9 / 17.6); wider tiles gain nothing (700 rows x 3584 x
  // 14336, 160 wide: 69.1 / 69.3 us)
  d.atoms = d.bn <= 128 ? 2 : 1;
  d.stages = pk::stage_room<O>() / (d.atoms * (pk::A_BLOCK + d.bn / 2 * BK * 2));
  if (d.stages > pk::MAX_STAGES) d.stages = pk::MAX_STAGES;
  const CUtensorMapSwizzle osw = sizeof(O) == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (encode_operand<T>(&d.tmX, a.x, a.M, a.K, a.ldx, 128) != QI_OK ||
      encode_operand<T>(&d.tmW, a.w, (wide ? 2ll : 1ll) * a.N, a.K, a.ldw, d.bn / 2) != QI_OK ||
      encode<O>(&d.tmO, a.out, a.M, a.N, a.ldo, 32, 32, osw) != QI_OK ||
      (a.residual && encode<O>(&d.tmR, a.residual, a.M, a.N, a.ldr, 32, 32, osw) != QI_OK))
    return QI_ERR_CUDA;
  static unsigned long long attr_done = 0;
  const auto fn = linear16_pair_kernel<T, O, SUMS>;
  if (SUMS) {
    // The register split counts on LAUNCH_REGS per thread at launch: with fewer,
    // the epilogue warps would wait for theirs without end.  A build that gave the
    // kernel another number is refused
    static int checked = 0;
    if (!__atomic_load_n(&checked, __ATOMIC_ACQUIRE)) {
      cudaFuncAttributes fa;
      if (cudaFuncGetAttributes(&fa, reinterpret_cast<const void*>(fn)) != cudaSuccess) {
        cudaGetLastError();
        return QI_ERR_CUDA;
      }
      if (fa.numRegs != pk::LAUNCH_REGS) return QI_ERR_UNSUPPORTED;
      __atomic_store_n(&checked, 1, __ATOMIC_RELEASE);
    }
  }
  if (smem_optin(reinterpret_cast<const void*>(fn), pk::SMEM_BYTES, &attr_done) != QI_OK) return QI_ERR_CUDA;
  const int tiles = d.tiles_m * d.tiles_n;
  return launch16(fn, 2u * (tiles < clusters ? tiles : clusters), pk::THREADS, pk::SMEM_BYTES, d, stream);
}

template <typename T, typename O, int G, int R, bool WIDE>
int launch_rows(const Linear16Args& a, cudaStream_t stream) {
  constexpr int COLS = WIDE ? 16 : 16 * R;
  constexpr int smem = rk::WARPS * 8 * G * (16 * R + 4) * 4;
  static_assert(smem <= 48 * 1024, "shared memory that needs no opt-in");
  return launch16(linear16_rows_kernel<T, O, G, R, WIDE>, static_cast<unsigned>((a.N + COLS - 1) / COLS), rk::THREADS, smem, a,
                  stream);
}

template <typename T, typename O>
int launch_typed(const Linear16Args& a, cudaStream_t stream) {
  // The rows kernel where it is the faster one (us, rows / pair kernel, FP32 or
  // 16-bit out): N 4608, K 3584: 1 row 10.4 / 16.7, 16 rows 14.0 / 16.8, 24 rows
  // 18.8 / 15.6; N = K = 512: 1 row 2.6 / 4.9; SwiGLU, N 14336, K 3584: 1 row
  // 45 / 46, 8 rows 50 / 46 (but 2.6 / 4.9 at small sizes), 16 rows 62 / 46.
  if (a.act == QI_ACT_SWIGLU) {
    if (a.M <= 8) return launch_rows<T, O, 1, 2, true>(a, stream);
  } else if (a.M <= 16) {
    return a.M <= 8 ? launch_rows<T, O, 1, 1, false>(a, stream) : launch_rows<T, O, 2, 1, false>(a, stream);
  }
  L16Dev d;
  memset(&d, 0, sizeof(d));
  d.bias = a.bias;
  d.gate = a.gate;
  d.residual = a.residual;
  d.M = a.M;
  d.N = a.N;
  d.K = a.K;
  d.act = a.act;
  if (a.K > pk::sums_min_k<T, O>(a.act == QI_ACT_SWIGLU)) return launch_pair16<T, O, true>(a, d, stream, device_num_sms());
  return launch_pair16<T, O, false>(a, d, stream, device_num_sms());
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
