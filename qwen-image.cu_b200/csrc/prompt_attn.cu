// prompt_attn.cu -- softmax attention over packed sequences with grouped heads,
// on the 5th-generation tensor cores.
//
// For one query row with products r_j = q.k_j over the keys it sees and sc =
// scale log2(e): running maximum m of the r_j and sum l (FP32), weights
// 2^(sc (r_j - m)) rounded to the 16-bit type, O = sum of weights times v in FP32,
// out = O / l.
//
// Work split.  The heads of a group read the same keys, so a 128-row query tile
// holds T = 128 / P tokens of P heads of one group (P = the group's size up to
// 128): row = token in tile * P + head.  K and V are read once for the group,
// and a causal tile spans few positions, so little of its last key block is
// masked.  A CTA runs NT tiles over one K / V stream; with few tiles the keys
// are also split, by the actual lengths (every CTA works out the same division
// from them), and a second kernel joins the parts.
//
// A CTA's warps: 0 TMA producer, 1 MMA issuer, 2-3 the V guard (below), then a
// warpgroup of softmax threads per tile (thread = row = TMEM lane).  Per 128-key
// block and tile: S = Q K^T into TMEM (kind::f16, FP32), the softmax thread reads
// its row, writes the weights as packed 16-bit over columns 0-63 of S, and
// O += P V takes P from TMEM and V (token-major) from shared memory.  Two tiles'
// S and O fill TMEM, so a tile's next S waits for its P V, and the other tile's
// products run under its softmax.
//
// Measured (device time of calls in one graph; back to back, where the power cap
// sets the clock, in brackets): 8192 causal tokens, 28 heads on 4 of 128: 431-434 us
// (500), 1110 TFLOP/s, tensor cores busy for 53% of the time; 24 heads x 2 x 4352
// keys: 428-473 us (495).  A key block of two tiles takes some 4000 clocks, of which
// its products and its exponentials each need 2048 and overlap: bound by the chain S
// -> softmax -> P V of each tile, a thread per row with two warps per scheduler to
// hide its latencies.  (The two-tile kernels spill a few registers: 68 bytes stored
// and 144 loaded per thread at heads of 128, 28 and 100 at 64.)  One token each
// against 16 caches of up to 4096: 24.2-25.9 us, one cache of 30000: 24.1-25.5 us, of
// which reading K and V takes 9: the rest is set-up, the first loads' latency and
// the joining launch.
//
// Sums.  The tensor cores truncate O every 16 keys.  Off by up to 6e-9 of sum p |v|
// per key of a split: 3e-5 at 4096 keys with v of one sign, 1.4e-3 at 262144 that are
// not split (a half step of FP16 is 4.9e-4, of BF16 3.9e-3).  TMEM is full with two
// tiles of heads of 128, so there is no room for a second sum.
//
// V guard.  A masked weight is 0, but 0 times a NaN or infinity of v is NaN: in
// blocks with masked keys (the last ones) the guard clears the V rows that no
// row of the CTA sees and, in rows that only some see, the elements that are not
// finite, before P V reads them.  It notes from which key on those are seen, and
// the epilogue gives exactly the rows that see them the NaN or infinity.
#include "qi_internal.h"
#include "sm100.cuh"

#include <limits.h>
#include <math.h>

#include <type_traits>

namespace qi {
namespace {

__device__ int g_prompt_attn_err;  // set by a bounded wait that gave up (prompt_attention_take_error)

constexpr int BQ = 128, BKV = 128;
constexpr int CACHED_SEQS = 256;  // sequences whose ranges a CTA keeps in shared memory
constexpr int HALF_BYTES = 128 * 128;  // 128 rows x 64 elements: one swizzled box column

template <int DH, int NT>
struct Cfg {
  static constexpr int NH = DH / 64;                                // 64-element halves of a head
  static constexpr int KS = NT == 2 && DH == 128 ? 2 : 3, VS = 2;   // K and V stages
  static constexpr int THREADS = 128 + 128 * NT;
  static constexpr int MIN_CTAS = NT == 1 && DH == 64 ? 2 : 1;
  static constexpr int LAUNCH_REGS = NT == 2 ? 168 : (MIN_CTAS == 2 ? 128 : 256);
  static constexpr int PRODUCER_REGS = NT == 2 ? 88 : 64, SOFTMAX_REGS = NT == 2 ? 208 : 192;
  static_assert(128 * PRODUCER_REGS + 128 * NT * SOFTMAX_REGS <= THREADS * LAUNCH_REGS, "register split exceeds the launch");
  static constexpr int TILE = NH * HALF_BYTES;  // Q tile, K block or V block
  static constexpr int OFF_K = NT * TILE, OFF_V = OFF_K + KS * TILE, OFF_X = OFF_V + VS * TILE;
  static constexpr int SMEM = 1024 + OFF_X + 2048 + 16 * CACHED_SEQS;
  static constexpr int TMEM_COLS = 256 * NT;  // S of tile t at 128 t, O at 128 (NT + t)
};

struct alignas(64) PromptAttnDev {
  CUtensorMap tmQ, tmK, tmV, tmO;
  PromptAttnArgs a;
  int P, T, packs;   // heads per tile row group, tokens per tile, tiles' head packs per kv head
  int items;         // work items per head pack at most: (unit of NT tiles, split of its keys) (gridDim.x)
  int splits;        // splits of a sequence's keys at most
  float sc;          // |scale| log2(e)
  float step;        // 8 / sc: what a row's maximum grows by before it moves
  uint32_t negate;   // scale < 0: instruction descriptor bit 13 (negate A) for Q K^T
  float* part;       // splits > 1: [splits][total_q * heads][DH] normalised partial outputs
  float2* ml;        // splits > 1: [splits][total_q * heads] (m, l), m before scaling
  int* used;         // splits > 1: [total_q * heads] splits that hold the row's keys
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Products with sc, which may be subnormal: without the flushing to zero that
// this build's own multiplications have.
__device__ __forceinline__ float mul_sub(float a, float b) {
  float y;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float fma_sub(float a, float b, float c) {
  float y;
  asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint64_t f2fma_sub(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ void settle(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = global_timer_ns();
  while (!mbar_try_wait(bar, parity) && global_timer_ns() - t0 < kWaitLimitNs / 4) {
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Last key (relative to the sequence) that token i of the sequence sees, or -1.
__device__ __forceinline__ int last_seen(int i, int lq, int lk, int causal) {
  return causal ? max(min(i + lk - lq, lk - 1), -1) : lk - 1;
}

// A sequence's ranges, clipped to the tensors: (q0, Lq, k0, Lk).
__device__ __forceinline__ int4 sequence(const PromptAttnArgs& a, int b) {
  const int q0 = a.q_begin[b], q1 = a.q_end[b], k0 = a.k_begin[b], k1 = a.k_end[b];
  int4 p;
  p.x = min(max(q0, 0), a.total_q);
  p.y = min(max(q1, p.x), a.total_q) - p.x;
  p.z = min(max(k0, 0), a.total_k);
  p.w = min(max(k1, p.z), a.total_k) - p.z;
  return p;
}
// A work item: the unit-th step of a sequence's tokens, the split-th part of its keys.
struct Place {
  int q0, lq, k0, lk;
  int unit, split;
};
// Units of `step` tokens of a sequence, and key blocks of its last one.
__device__ __forceinline__ int units_of(int4 p, int step) { return (p.y + step - 1) / step; }
__device__ __forceinline__ int blocks_of(int4 p, int causal) {
  return p.y > 0 ? (last_seen(p.y - 1, p.y, p.w, causal) + BKV) / BKV : 0;
}
__device__ __forceinline__ int splits_of(int blocks, int chunk) { return max(1, (blocks + chunk - 1) / chunk); }

// Which work item CTA `idx` of a head pack takes, and the key blocks per split.
// Called by one whole warp; leaves the first CACHED_SEQS sequences in `seqs`.
// False when there are fewer items.
//
// Splits: the smallest chunk of key blocks that keeps all sequences' items within
// args.items (whole waves of CTAs) and a sequence's splits within args.splits,
// worked out from the lengths by every CTA alike.
// Order (BY_INDEX): a causal sequence's later units see more keys, so the units of
// all sequences go by their index, the last first.
template <bool BY_INDEX>
__device__ __forceinline__ bool schedule(const PromptAttnDev& d, int step, int idx, int4* seqs, int& chunk, Place& out) {
  const PromptAttnArgs& a = d.a;
  const int lane = threadIdx.x & 31;
  int most = 0, most_units = 0, u0 = 0, n0 = 0;  // u0, n0: units and blocks of sequence `lane`
  float work = 0.0f;
  for (int b = lane; b < a.batch; b += 32) {
    const int4 p = sequence(a, b);
    if (b < CACHED_SEQS) seqs[b] = p;
    const int u = units_of(p, step), n = blocks_of(p, a.causal);
    if (b == lane) {
      u0 = u;
      n0 = n;
    }
    most = max(most, n);
    most_units = max(most_units, u);
    work += static_cast<float>(u) * static_cast<float>(n);
  }
  __syncwarp();
  auto seq = [&](int b) { return b < CACHED_SEQS ? seqs[b] : sequence(a, b); };
  auto take = [&](int4 p, int unit, int split) {
    out.q0 = p.x;
    out.lq = p.y;
    out.k0 = p.z;
    out.lk = p.w;
    out.unit = unit;
    out.split = split;
  };
  chunk = INT_MAX / 2;
  if (BY_INDEX && d.splits == 1 && a.causal) {
    most_units = __reduce_max_sync(0xffffffffu, most_units);
    auto count = [&](int unit) {  // units with this index or a higher one
      int n = max(0, u0 - unit);
      for (int b = lane + 32; b < a.batch; b += 32) n += max(0, units_of(seq(b), step) - unit);
      return __reduce_add_sync(0xffffffffu, n);
    };
    if (idx >= count(0)) return false;
    int lo = 0, hi = most_units;  // count(lo) > idx >= count(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (count(mid) > idx)
        lo = mid;
      else
        hi = mid;
    }
    int r = idx - count(lo + 1);  // the r-th sequence that has a unit lo
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      const int u = b0 == 0 ? u0 : (b0 + lane < a.batch ? units_of(seq(b0 + lane), step) : 0);
      unsigned m = __ballot_sync(0xffffffffu, u > lo);
      if (r >= __popc(m)) {
        r -= __popc(m);
        continue;
      }
      for (; r > 0; --r) m &= m - 1;
      take(seq(b0 + __ffs(m) - 1), lo, 0);
      return true;
    }
    return false;
  }
  if (d.splits > 1) {
    most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
    for (int i = 16; i > 0; i /= 2) work += __shfl_xor_sync(0xffffffffu, work, i);
    chunk = max(max(2, (most + d.splits - 1) / d.splits), static_cast<int>(ceilf(fminf(work / d.items, static_cast<float>(most)))));
    while (chunk < most) {
      int n = u0 * splits_of(n0, chunk);
      for (int b = lane + 32; b < a.batch; b += 32) {
        const int4 p = seq(b);
        n += units_of(p, step) * splits_of(blocks_of(p, a.causal), chunk);
      }
      if (__reduce_add_sync(0xffffffffu, n) <= d.items) break;
      chunk += max(1, chunk / 8);
    }
  }
  // the sequences' items follow one another
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    int n = u0, s = n0;
    if (b0 > 0) {
      const int4 p = b0 + lane < a.batch ? seq(b0 + lane) : make_int4(0, 0, 0, 0);
      n = units_of(p, step);
      s = blocks_of(p, a.causal);
    }
    if (d.splits > 1) {
      s = splits_of(s, chunk);
      n *= s;
    } else {
      s = 1;
    }
    int sum = n;  // inclusive prefix sum over the lanes
#pragma unroll
    for (int i = 1; i < 32; i *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, sum, i);
      if (lane >= i) sum += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, idx < sum);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int r = idx - __shfl_sync(0xffffffffu, sum - n, src), sp = __shfl_sync(0xffffffffu, s, src);
      take(seq(b0 + src), r / sp, r % sp);
      return true;
    }
    idx -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

template <typename T>
constexpr uint32_t idesc(int M, int N, bool b_mn) {
  return idesc_f16(M, N, false, b_mn) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u);
}

template <typename T, int DH, int NT>
__global__ void __launch_bounds__(Cfg<DH, NT>::THREADS, Cfg<DH, NT>::MIN_CTAS)
    prompt_attn_kernel(const __grid_constant__ PromptAttnDev args) {
  using C = Cfg<DH, NT>;
  constexpr int NH = C::NH, KS = C::KS, VS = C::VS, TILE = C::TILE;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + C::OFF_K;
  uint8_t* sV = smem + C::OFF_V;
  int* bad = reinterpret_cast<int*>(smem + C::OFF_X);  // [3][DH] first key with NaN / +inf / -inf in a dimension
  uint64_t* q_full = reinterpret_cast<uint64_t*>(bad + 3 * 128);
  uint64_t* k_full = q_full + 1;       // [KS]
  uint64_t* k_empty = k_full + KS;     // [KS]
  uint64_t* v_full = k_empty + KS;     // [VS]
  uint64_t* v_ready = v_full + VS;     // [VS] the V guard has passed the block (2 warps)
  uint64_t* v_empty = v_ready + VS;    // [VS]
  uint64_t* s_full = v_empty + VS;     // [NT] QK of the tile's current block complete
  uint64_t* s_loaded = s_full + NT;    // [NT] the tile's S is in registers (4 warps; one-tile CTAs)
  uint64_t* p_half = s_loaded + NT;    // [NT][2] half h of the tile's P is in TMEM (4 warps)
  uint64_t* o_final = p_half + 2 * NT; // [NT] the tile's last PV complete
  uint64_t* drain = o_final + NT;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* any_bad = const_cast<int*>(abort_flag) + 1;
  Place* place = reinterpret_cast<Place*>(any_bad + 1);
  int* found = reinterpret_cast<int*>(place + 1);
  int* chunk_slot = found + 1;
  int4* seqs = reinterpret_cast<int4*>(smem + C::OFF_X + 2048);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PromptAttnArgs& a = args.a;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < KS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < VS; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ready[i], 2);
      mbar_init(&v_empty[i], 1);
    }
    for (int t = 0; t < NT; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_loaded[t], 4);
      mbar_init(&p_half[2 * t], 4);
      mbar_init(&p_half[2 * t + 1], 4);
      mbar_init(&o_final[t], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *any_bad = 0;
    fence_mbar_init();
    tma_prefetch_desc(&args.tmQ);
    tma_prefetch_desc(&args.tmK);
    tma_prefetch_desc(&args.tmV);
    tma_prefetch_desc(&args.tmO);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 2)
    for (int i = lane; i < 3 * DH; i += 32) bad[i] = INT_MAX;
  grid_dependency_wait();
  if (warp == 0) {
    Place p = {};
    int c;
    const bool ok = schedule<NT == 2>(args, NT * args.T, blockIdx.x, seqs, c, p);
    if (lane == 0) {
      *place = p;
      *found = ok;
      *chunk_slot = c;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  launch_dependents();  // after the allocation: a dependent CTA on this SM gets what is left of TMEM
  const uint32_t tmem = *tmem_slot;
  const Place pl = *place;
  const int chunk = *chunk_slot;
  const int tok0 = pl.unit * NT * args.T;  // first token of the unit in its sequence
  // key blocks [jb, je[t]) of tile t in this split; n[t] of them
  int n[NT], nkb[NT], nmax = 0;
  const int jb = pl.split * chunk;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int first = tok0 + t * args.T, lim = last_seen(min(first + args.T, pl.lq) - 1, pl.lq, pl.lk, a.causal);
    nkb[t] = *found && first < pl.lq ? (lim + BKV) / BKV : 0;  // lim = -1: none
    const int je = min(nkb[t], jb + chunk);
    n[t] = max(0, je - jb);
    nmax = max(nmax, n[t]);
  }
  // keys past the first token's last are masked for some row, past the unit's
  // last token's for all
  const int lim_first = last_seen(tok0, pl.lq, pl.lk, a.causal);
  const int lim_unit = last_seen(min(tok0 + NT * args.T, pl.lq) - 1, pl.lq, pl.lk, a.causal);
  const int y = blockIdx.y, hk = y / args.packs;

  if (warp < 4) {
    if (C::LAUNCH_REGS < 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::PRODUCER_REGS));
    if (warp == 0) {
      // -------------------------------------------------------------- producer
      if (lane == 0 && nmax > 0) {
        bool ok = true;
        uint32_t kmask = 0, kpar = 0, vmask = 0, vpar = 0;
        mbar_expect_tx(q_full, NT * NH * args.T * args.P * 128);
        for (int t = 0; t < NT; ++t)
          for (int h = 0; h < NH; ++h)
            tma_load_4d(sQ + t * TILE + h * HALF_BYTES, &args.tmQ, 64 * h, 0, pl.q0 + tok0 + t * args.T, y, q_full);
        for (int i = 0; i < nmax && ok; ++i) {
          const int ks = i % KS, vs = i % VS, row = pl.k0 + (jb + i) * BKV;
          const uint32_t kp = (i / KS) & 1, vp = (i / VS) & 1;
          if (!mbar_wait(&k_empty[ks], kp ^ 1u, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&k_full[ks], TILE);
          for (int h = 0; h < NH; ++h) tma_load_3d(sK + ks * TILE + h * HALF_BYTES, &args.tmK, 64 * h, hk, row, &k_full[ks]);
          kmask |= 1u << ks;
          kpar = (kpar & ~(1u << ks)) | (kp << ks);
          if (!mbar_wait(&v_empty[vs], vp ^ 1u, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&v_full[vs], TILE);
          for (int h = 0; h < NH; ++h) tma_load_3d(sV + vs * TILE + h * HALF_BYTES, &args.tmV, 64 * h, hk, row, &v_full[vs]);
          vmask |= 1u << vs;
          vpar = (vpar & ~(1u << vs)) | (vp << vs);
        }
        if (!ok) {  // let the copies already issued land before the CTA exits
          *abort_flag = 1;
          atomicCAS(&g_prompt_attn_err, 0, kErrTimeoutProducer);
          settle(q_full, 0);
          for (int s = 0; s < KS; ++s)
            if (kmask & (1u << s)) settle(&k_full[s], (kpar >> s) & 1u);
          for (int s = 0; s < VS; ++s)
            if (vmask & (1u << s)) settle(&v_full[s], (vpar >> s) & 1u);
        }
      }
    } else if (warp == 1) {
      // -------------------------------------------------------------- MMA issuer
      if (nmax > 0) {
        // every lane waits; the vote keeps the warp converged for elect.sync
        auto wait_all = [&](uint64_t* bar, uint32_t parity) {
          return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
        };
        const uint32_t id_qk = idesc<T>(BQ, BKV, false) | args.negate, id_qk64 = idesc<T>(BQ, 64, false) | args.negate;
        const uint32_t id_pv = idesc<T>(BQ, DH, true);
        const uint64_t qd0 = umma_desc_sw128(smem_u32(sQ), 16, 1024), kd0 = umma_desc_sw128(smem_u32(sK), 16, 1024);
        const uint64_t vd0 = umma_desc_sw128(smem_u32(sV), HALF_BYTES, 1024);
        // S_t = Q_t K^T: all 128 keys, or keys 64 hh .. of them (columns 64 hh ..)
        auto qk = [&](int t, int ks) {
#pragma unroll
          for (int k = 0; k < DH / 16; ++k) {
            const uint64_t off = (k / 4) * (HALF_BYTES >> 4) + 2 * (k % 4);
            mma_f16_ss_elect(tmem + 128 * t, qd0 + static_cast<uint64_t>((t * TILE) >> 4) + off,
                             kd0 + static_cast<uint64_t>((ks * TILE) >> 4) + off, id_qk, k > 0 ? 1u : 0u);
          }
        };
        auto qk_half = [&](int t, int ks, int hh) {
#pragma unroll
          for (int k = 0; k < DH / 16; ++k) {
            const uint64_t off = (k / 4) * (HALF_BYTES >> 4) + 2 * (k % 4);
            mma_f16_ss_elect(tmem + 128 * t + 64 * hh, qd0 + static_cast<uint64_t>((t * TILE) >> 4) + off,
                             kd0 + static_cast<uint64_t>((ks * TILE + hh * (HALF_BYTES / 2)) >> 4) + off, id_qk64,
                             k > 0 ? 1u : 0u);
          }
        };
        // O_t += P_t V over keys 64 h .. of the block
        auto pv_half = [&](int t, int vs, int i, int h) {
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            const int kk = 4 * h + k4;
            mma_f16_ts_elect(tmem + 128 * (NT + t), tmem + 128 * t + 8 * kk,
                             vd0 + static_cast<uint64_t>((vs * TILE) >> 4) + 128 * kk, id_pv, (i > 0 || kk > 0) ? 1u : 0u);
          }
        };
        bool ok = wait_all(q_full, 0) && wait_all(&k_full[0], 0);
        if (ok) {
          tc_fence_after();
          for (int t = 0; t < NT; ++t) {
            if (n[t] == 0) continue;
            qk(t, 0);
            mma_commit_elect(&s_full[t]);
          }
          mma_commit_elect(&k_empty[0]);
        }
        // P occupies half of S_t's columns, so the next block's product goes
        // behind P_t V; a CTA's MMAs run in issue order.  With two tiles it is
        // one N = 128 product (the other tile's work fills the time; 8192 causal
        // tokens: 454 us against 484 us with halves).  With one, its upper half
        // of keys, whose columns never hold P, goes ahead as soon as S_t has been
        // read (N = 64 products re-read Q twice as often, but nothing else wants
        // the tensor cores: 16 caches of up to 4096, 34.6 against 35.7 us).
        constexpr bool EARLY = NT == 1;
        for (int i = 0; i < nmax && ok; ++i) {
          const int vs = i % VS, ks = (i + 1) % KS;
          const uint32_t vp = (i / VS) & 1, kp = ((i + 1) / KS) & 1;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (!ok || i >= n[t]) continue;
            const bool more = i + 1 < n[t];
            // the last tile that still uses this V block / the next K block
            const bool last_v = t == NT - 1 || i >= n[NT - 1], last_k = t == NT - 1 || i + 1 >= n[NT - 1];
            if (more && EARLY) {
              ok = wait_all(&s_loaded[t], i & 1) && wait_all(&k_full[ks], kp);
              if (!ok) break;
              tc_fence_after();
              qk_half(t, ks, 1);
            }
            ok = wait_all(&p_half[2 * t], i & 1) && wait_all(&v_ready[vs], vp);
            if (!ok) break;
            tc_fence_after();
            pv_half(t, vs, i, 0);
            ok = wait_all(&p_half[2 * t + 1], i & 1);
            if (!ok) break;
            tc_fence_after();
            pv_half(t, vs, i, 1);
            if (!more) mma_commit_elect(&o_final[t]);
            if (last_v) mma_commit_elect(&v_empty[vs]);
            if (more) {
              if (EARLY) {
                qk_half(t, ks, 0);
              } else {
                ok = wait_all(&k_full[ks], kp);
                if (!ok) break;
                tc_fence_after();
                qk(t, ks);
              }
              mma_commit_elect(&s_full[t]);
              if (last_k) mma_commit_elect(&k_empty[ks]);
            }
          }
        }
        if (!ok && lane == 0) {
          *abort_flag = 1;
          atomicCAS(&g_prompt_attn_err, 0, kErrTimeoutMma);
        }
        __syncwarp();
        mma_commit_elect(drain);  // every MMA issued above completes before TMEM is released
        settle(drain, 0);
      }
    } else {
      // -------------------------------------------------------------- V guard
      constexpr uint32_t EXP = std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;  // NaN or infinity: all set
      bool ok = true;
      for (int i = 0; i < nmax && ok; ++i) {
        const int vs = i % VS, key0 = (jb + i) * BKV;
        ok = __all_sync(0xffffffffu, mbar_wait(&v_full[vs], (i / VS) & 1, abort_flag));
        if (!ok) break;
        if (key0 + BKV - 1 > lim_first) {
          // 16-byte pieces of the rows nobody sees (cleared), and before them of
          // the rows that some see and some do not (checked)
          const int scan0 = max(lim_first + 1 - key0, 0) * 8, zero0 = min(max(lim_unit + 1 - key0, 0), BKV) * 8;
          uint8_t* blk = sV + vs * TILE;
          for (int c = zero0 + (warp - 2) * 32 + lane; c < BKV * 8; c += 64)
#pragma unroll
            for (int h = 0; h < NH; ++h) *reinterpret_cast<uint4*>(blk + h * HALF_BYTES + c * 16) = make_uint4(0u, 0u, 0u, 0u);
          for (int c = scan0 + (warp - 2) * 32 + lane; c < zero0; c += 64)
#pragma unroll
            for (int h = 0; h < NH; ++h) {
              uint8_t* p = blk + h * HALF_BYTES + c * 16;
              const uint4 v = *reinterpret_cast<const uint4*>(p);
              const uint32_t u[4] = {v.x, v.y, v.z, v.w};
              bool any = false;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                any |= ((u[e] & EXP) == EXP) | ((u[e] & (EXP << 16)) == (EXP << 16));
              if (any) {
                uint16_t* q = reinterpret_cast<uint16_t*>(p);
                for (int e = 0; e < 8; ++e) {
                  const uint32_t w = q[e];
                  if ((w & EXP) != EXP) continue;
                  const int kind = (w & (0x7FFFu ^ EXP)) ? 0 : (w & 0x8000u ? 2 : 1);
                  atomicMin(&bad[kind * DH + h * 64 + ((c & 7) ^ ((c >> 3) & 7)) * 8 + e], key0 + (c >> 3));
                  q[e] = 0;
                  *any_bad = 1;
                }
              }
            }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ready[vs]);
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        atomicCAS(&g_prompt_attn_err, 0, kErrTimeoutSoftmax);
      }
    }
  } else {
    if (C::LAUNCH_REGS < 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
    // ---------------------------------------------------------------- softmax
    const int t = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const int my_n = NT == 1 || t == 0 ? n[0] : n[NT - 1], my_nkb = NT == 1 || t == 0 ? nkb[0] : nkb[NT - 1];
    const int tok = row / args.P, i_tok = tok0 + t * args.T + tok;  // token in its sequence
    const bool valid = *found && tok < args.T && i_tok < pl.lq;
    // rows that are no query (their results go nowhere) do not ask for masking
    const int lim = valid ? last_seen(i_tok, pl.lq, pl.lk, a.causal) : lim_unit;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_tm = tmem + lane_off + 128 * t, o_tm = tmem + lane_off + 128 * (NT + t);
    // FP16 weights are kept in 2^7 .. 2^15 for the largest so that small ones
    // stay clear of the subnormals; the factor is in l too
    constexpr float LIFT = std::is_same<T, __half>::value ? 7.0f : 0.0f;
    // scores in base 2 up to which sc m may be rounded (off by 2^-16 at most)
    constexpr float FAR = 256.0f;
    const uint64_t sc2 = f2pack(args.sc, args.sc);
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int i = 0; i < my_n; ++i) {
      const bool w = mbar_wait(&s_full[t], i & 1, abort_flag);
      if (!__all_sync(0xffffffffu, w)) { ok = false; break; }
      tc_fence_after();
      uint32_t r[BKV];
#pragma unroll
      for (int c = 0; c < BKV; c += 32) tmem_ld32(s_tm + c, *reinterpret_cast<uint32_t(*)[32]>(r + c));
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < BKV; c += 32) tmem_reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(r + c));
      if (NT == 1) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_loaded[t]);
      }
      const int key0 = (jb + i) * BKV, seen = lim - key0;  // keys 0 .. seen of the block are seen
      float alpha = 1.0f;
      uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
      auto block = [&](auto masked_tag) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        if (MASKED) {
#pragma unroll
          for (int c = 0; c < BKV; ++c)
            if (c > seen) r[c] = 0xFF800000u;  // -inf: weight 0
        }
        float mx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = __uint_as_float(r[e]);
#pragma unroll
        for (int c = 4; c < BKV - 4; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(r[c + e]), __uint_as_float(r[c + e + 4]));
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(r[BKV - 4 + e]));
        const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
        // Lazy rescale: the maximum used moves only when the row's grows by more
        // than 8 in base 2 (weights stay <= 2^8); O and l move with it
        const float m_new = fmaxf(m, top);
        const bool grow = m_new - m > args.step;
        if (grow) {
          alpha = ex2(mul_sub(m - m_new, args.sc));
          m = m_new;
        }
        if (i > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
          for (int c = 0; c < DH; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_tm + c, o);
            tmem_ld_wait();
            tmem_reg_fence32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(o_tm + c, o);
          }
        }
        // Exponents sc (r - m): exact differences near the maximum, whatever its
        // size.  Or in one step, sc r - sc m, where rounding sc m is no error worth
        // minding.  With two tiles the first form is the faster one (8192 causal
        // tokens 432 against 449 us), with one the second (16 single tokens 25.6
        // against 24.2).  Nothing seen yet: every weight is 0
        const float base = m == -INFINITY ? 0.0f : fma_sub(-m, args.sc, LIFT);
        auto weights = [&](auto exact_tag) {
          constexpr bool EXACT = decltype(exact_tag)::value;
          const float off = !EXACT ? base : (m == -INFINITY ? 0.0f : -m);
          const uint64_t off2 = f2pack(off, off), lift2 = f2pack(LIFT, LIFT);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pk[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const int k = 64 * h + 2 * c;
              const uint64_t r2 = f2pack(__uint_as_float(r[k]), __uint_as_float(r[k + 1]));
              float p0, p1;
              f2unpack(EXACT ? f2fma_sub(f2add(r2, off2), sc2, lift2) : f2fma_sub(r2, sc2, off2), p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
              sum2[c & 3] = f2add(sum2[c & 3], f2pack(p0, p1));
              pk[c] = pack16<T>(p0, p1);
            }
            tmem_st32(s_tm + 32 * h, pk);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_half[2 * t + h]);
          }
        };
        if (NT == 2 || __builtin_expect(__any_sync(0xffffffffu, valid && fabsf(base) > FAR), 0))
          weights(std::true_type{});
        else
          weights(std::false_type{});
      };
      if (__any_sync(0xffffffffu, seen < BKV - 1))
        block(std::true_type{});
      else
        block(std::false_type{});
      float a0, a1;
      f2unpack(f2add(f2add(sum2[0], sum2[1]), f2add(sum2[2], sum2[3])), a0, a1);
      l = l * alpha + (a0 + a1);
    }
    // a tile without keys stages zeros where its Q may still be on its way, for
    // the other tile's sake (the producer brings both tiles' Q)
    if (ok && nmax > 0) ok = __all_sync(0xffffffffu, mbar_wait(my_n > 0 ? &o_final[t] : q_full, 0, abort_flag));
    // splits of this tile that hold keys; with one the output is final
    const int used = splits_of(my_nkb, chunk);
    // (two tiles: one-tile CTAs end sooner without a bulk store's round trip.
    // Packed prompts 76 / 83 us with / without it, chunks behind caches 42 / 39)
    const bool all_rows = NT == 2 && used == 1 && pl.split == 0 && *found && tok0 + (t + 1) * args.T <= pl.lq;
    auto tile_sync = [&]() {  // the tile's four warps
      if (t == 0)
        asm volatile("bar.sync 1, 128;" ::: "memory");
      else
        asm volatile("bar.sync 2, 128;" ::: "memory");
    };
    if (!ok) {
      if (lane == 0) {
        *abort_flag = 1;
        atomicCAS(&g_prompt_attn_err, 0, kErrTimeoutSoftmax);
      }
      __syncwarp();
      if (all_rows) tile_sync();  // the tile's other warps may be waiting there
    } else {
      // ---------------------------------------------------------------- epilogue
      tc_fence_after();
      const bool mine = valid && pl.split < used;
      const float rl = l == 0.0f ? 0.0f : 1.0f / l;  // NaN stays NaN
      const int head = y * args.P + row % args.P;
      const long long qrow = pl.q0 + i_tok, slot = qrow * a.heads + head;
      const long long part_rows = static_cast<long long>(a.total_q) * a.heads;
      float* part = args.part + (static_cast<long long>(pl.split) * part_rows + slot) * DH;
      const bool patch = *any_bad != 0;
      // the tile's Q is no longer read: its memory stages the outputs in Q's
      // layout (pieces of a row swizzled)
      uint8_t* stage = sQ + t * TILE + row * 128;
      if (my_n > 0) {
#pragma unroll 1
        for (int h = 0; h < NH; ++h) {
          uint32_t o[64];
          __syncwarp();
          tmem_ld32(o_tm + 64 * h, *reinterpret_cast<uint32_t(*)[32]>(o));
          tmem_ld32(o_tm + 64 * h + 32, *reinterpret_cast<uint32_t(*)[32]>(o + 32));
          tmem_ld_wait();
          tmem_reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(o));
          tmem_reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(o + 32));
          // l = 0: the row saw nothing
#pragma unroll
          for (int e = 0; e < 64; ++e) o[e] = l == 0.0f ? 0u : __float_as_uint(__uint_as_float(o[e]) * rl);
          if (patch && l != 0.0f) {
            const int* first = bad + 64 * h;
#pragma unroll
            for (int e = 0; e < 64; ++e) {
              const bool nan = first[e] <= lim, pos = first[DH + e] <= lim, neg = first[2 * DH + e] <= lim;
              if (nan | (pos & neg)) o[e] = 0x7FFFFFFFu;
              else if (pos | neg) o[e] = __float_as_uint(__uint_as_float(o[e]) + (pos ? INFINITY : -INFINITY));
              asm volatile("" ::: "memory");  // one element's loads at a time: this path is rare, registers are not
            }
          }
          if (used > 1) {
            if (mine) {
#pragma unroll
              for (int e = 0; e < 64; e += 4)
                *reinterpret_cast<uint4*>(part + 64 * h + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 64; e += 8)
              *reinterpret_cast<uint4*>(stage + h * HALF_BYTES + ((e >> 3) ^ (row & 7)) * 16) =
                  make_uint4(pack16<T>(__uint_as_float(o[e]), __uint_as_float(o[e + 1])),
                             pack16<T>(__uint_as_float(o[e + 2]), __uint_as_float(o[e + 3])),
                             pack16<T>(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5])),
                             pack16<T>(__uint_as_float(o[e + 6]), __uint_as_float(o[e + 7])));
          }
        }
      } else if (mine) {  // no keys at all
#pragma unroll
        for (int e = 0; e < DH; e += 8)
          *reinterpret_cast<uint4*>(stage + (e >> 6) * HALF_BYTES + (((e & 63) >> 3) ^ (row & 7)) * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      const unsigned rows_out = __ballot_sync(0xffffffffu, mine && used == 1);
      __syncwarp();
      if (all_rows) {  // the tile's tokens all exist: one copy per half, in Q's layout
        fence_proxy_async_smem();
        tile_sync();
        if (row == 0) {
          for (int h = 0; h < NH; ++h)
            if (64 * h < a.head_dim)
              tma_store_4d(&args.tmO, sQ + t * TILE + h * HALF_BYTES, 64 * h, 0, pl.q0 + tok0 + t * args.T, y);
          bulk_commit();
          bulk_wait_read<0>();
        }
      } else if (rows_out) {
        const long long at = qrow * a.o_row + head * a.o_head;
        const uint8_t* base = sQ + t * TILE + quarter * 32 * 128;
#pragma unroll 4
        for (int r4 = 0; r4 < 32; r4 += 4) {
          const int r = r4 + (lane >> 3), piece = lane & 7;
          const long long off = __shfl_sync(0xffffffffu, at, r);
          if (!((rows_out >> r) & 1u)) continue;
          T* out = static_cast<T*>(a.out) + off + piece * 8;
#pragma unroll
          for (int h = 0; h < NH; ++h)
            if (64 * h + piece * 8 < a.head_dim)
              *reinterpret_cast<uint4*>(out + 64 * h) =
                  *reinterpret_cast<const uint4*>(base + h * HALF_BYTES + r * 128 + (piece ^ (r & 7)) * 16);
        }
      }
      if (mine && pl.split == 0 && args.splits > 1) args.used[slot] = used;
      if (mine && used > 1) args.ml[static_cast<long long>(pl.split) * part_rows + slot] = make_float2(m, l);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Joins the splits of a row: out = sum_s w_s O_s / sum_s w_s, w_s = l_s 2^(sc (m_s - max m)).
// A CTA per token and 8 / per heads; `per` warps per head take its splits in
// turn, four dimensions per thread, and add up in warp order.  Rows whose tile
// had one split are final already.
struct JoinDev {
  void* out;
  long long o_row, o_head;
  const int* q_begin;
  const int* q_end;
  const float* part;
  const float2* ml;
  const int* used;
  int batch, total_q, heads, head_dim;
  int warps, splits;  // warps per head; splits the workspace holds
  float sc;
};
template <typename T, int DH>
__global__ void __launch_bounds__(256) prompt_attn_join_kernel(const __grid_constant__ JoinDev args) {
  constexpr int AHEAD = 6;
  __shared__ float4 part_o[8][32];
  __shared__ float2 part_w[8];
  grid_dependency_wait();
  launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = args.warps, wi = warp % per;
  const int qrow = blockIdx.x, head = blockIdx.y * (8 / per) + warp / per;
  const long long rows = static_cast<long long>(args.total_q) * args.heads;
  const long long slot = static_cast<long long>(qrow) * args.heads + head;
  // Read ahead of the look-up, to have one round trip to memory instead of
  // three: the row's split count, this warp's first (m, l) and, with few rows
  // (per > 1), partial outputs, all inside the workspace; what is past the
  // row's splits, or belongs to no sequence, means nothing and is not used.
  // The count is bounded: query ranges that overlap can ask for more items than
  // the grid has, and rows of those that are left out have no count
  const int used = head < args.heads ? min(args.used[slot], args.splits) : 0;
  float2 ml0 = make_float2(-INFINITY, 0.0f);
  if (head < args.heads && wi + lane * per < args.splits) ml0 = args.ml[(wi + static_cast<long long>(lane) * per) * rows + slot];
  float4 v0[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (per > 1 && head < args.heads && wi + i * per < args.splits && 4 * lane < DH)
      v0[i] = *reinterpret_cast<const float4*>(args.part + ((wi + static_cast<long long>(i) * per) * rows + slot) * DH + 4 * lane);
  bool found = false;
  for (int b0 = 0; b0 < args.batch && !found; b0 += 32) {
    bool hit = false;
    if (b0 + lane < args.batch) hit = qrow >= args.q_begin[b0 + lane] && qrow < args.q_end[b0 + lane];
    found = __any_sync(0xffffffffu, hit);
  }
  const bool work = found && head < args.heads && used > 1;
  // this warp's splits: wi, wi + per, ...; lane i holds the i-th's (m, l)
  const int mine = work && wi < used ? (used - wi + per - 1) / per : 0;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float total = 0.0f, top = -INFINITY;
  for (int i0 = 0; i0 < mine; i0 += 32) {
    const long long s = wi + static_cast<long long>(i0 + lane) * per;
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (i0 + lane < mine) ml = i0 == 0 ? ml0 : args.ml[s * rows + slot];
    float t = ml.y == 0.0f ? -INFINITY : ml.x;  // l = 0: this part saw nothing
#pragma unroll
    for (int d = 16; d > 0; d /= 2) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
    t = fmaxf(t, top);
    const float keep = top == -INFINITY ? 0.0f : ex2(mul_sub(top - t, args.sc));
    top = t;
    total *= keep;
    o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
    const float w_lane = ml.y == 0.0f ? 0.0f : ml.y * ex2(mul_sub(ml.x - top, args.sc));
    const int ahead = per > 1 && i0 == 0 ? min(mine, AHEAD) : 0;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float w = __shfl_sync(0xffffffffu, w_lane, i);
      if (i >= ahead || w == 0.0f || 4 * lane >= DH) continue;
      total += w;
      o = make_float4(o.x + w * v0[i].x, o.y + w * v0[i].y, o.z + w * v0[i].z, o.w + w * v0[i].w);
    }
#pragma unroll 4
    for (int i = ahead; i < min(mine - i0, 32); ++i) {
      const float w = __shfl_sync(0xffffffffu, w_lane, i);
      if (w == 0.0f || 4 * lane >= DH) continue;
      const float4 v = *reinterpret_cast<const float4*>(
          args.part + ((wi + static_cast<long long>(i0 + i) * per) * rows + slot) * DH + 4 * lane);
      total += w;
      o = make_float4(o.x + w * v.x, o.y + w * v.y, o.z + w * v.z, o.w + w * v.w);
    }
    total = __shfl_sync(0xffffffffu, total, 0);
  }
  if (per > 1) {
    part_o[warp][lane] = o;
    if (lane == 0) part_w[warp] = make_float2(top, total);
    __syncthreads();
    if (wi != 0) return;
    for (int i = 0; i < per; ++i) top = fmaxf(top, part_w[warp + i].x);
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    total = 0.0f;
    for (int i = 0; i < per; ++i) {
      const float2 tw = part_w[warp + i];
      if (tw.x == -INFINITY && tw.y == 0.0f) continue;
      const float k = ex2(mul_sub(tw.x - top, args.sc));
      const float4 v = part_o[warp + i][lane];
      total += k * tw.y;
      o = make_float4(o.x + k * v.x, o.y + k * v.y, o.z + k * v.z, o.w + k * v.w);
    }
  }
  if (!work || 4 * lane >= args.head_dim) return;
  const float r = total == 0.0f ? 0.0f : 1.0f / total;
  T* out = static_cast<T*>(args.out) + qrow * args.o_row + head * args.o_head + 4 * lane;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack16<T>(o.x * r, o.y * r), pack16<T>(o.z * r, o.w * r));
}

// ------------------------------------------------------------------ host
struct Plan {
  int P, T, packs, nt, splits, dh;
  long long items;
};

Plan plan_of(int heads, int kv_heads, int head_dim, int batch, int total_q, int max_k, int num_sms) {
  Plan p;
  const int G = heads / kv_heads;
  p.dh = head_dim <= 64 ? 64 : 128;
  p.P = G;
  while (p.P > BQ || G % p.P) --p.P;
  p.T = BQ / p.P;
  p.packs = G / p.P;
  const long long groups = heads / p.P;
  // One tile per CTA while those fit on the device at once (shorter calls) or
  // sequences fill no second one; two over one K / V stream beyond that.  One /
  // two tiles: a pair of short prompts 7.2 / 9.0 us, one token for each of 16
  // caches 24 / 27; packed prompts 107 / 78, 8192 causal tokens 714 / 453
  const long long ctas1 = (static_cast<long long>(total_q) / p.T + batch) * groups;
  p.nt = ctas1 <= num_sms || total_q < 2ll * p.T * batch ? 1 : 2;
  const long long units = static_cast<long long>(total_q) / (p.nt * p.T) + batch, ctas = units * groups;
  // Key splits while the units alone leave the device (two CTAs per SM with
  // heads of 64) short of work, or, one token each, of even work; at least two
  // blocks each.  More than 4 (2) x the CTAs it holds would only cost workspace.
  const long long slots = static_cast<long long>(num_sms) * (p.nt == 1 && p.dh == 64 ? 2 : 1);
  long long splits = (p.nt == 1 ? 4 : 2) * slots / ctas;
  const int blocks = max_k / BKV + (max_k % BKV != 0);
  if (splits > blocks / 2) splits = blocks / 2;
  p.splits = splits < 1 ? 1 : static_cast<int>(splits);
  const long long wave = slots / groups < 1 ? 1 : slots / groups;  // work items per head group that run at once
  p.items = p.splits > 1 ? (units + wave - 1) / wave * wave : units;
  return p;
}

int encode_heads(CUtensorMap* tm, int dtype, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                 const cuuint32_t* box) {
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = qi_encode_tiled(tm, dtype == QI_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                     rank, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? QI_OK : QI_ERR_CUDA;
}

template <typename A>
int launch_dependent(void (*fn)(const A), dim3 grid, int threads, int smem, const A& args, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
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

template <typename T, int DH, int NT>
int launch_tiles(const PromptAttnDev& d, cudaStream_t stream) {
  using C = Cfg<DH, NT>;
  static_assert(C::SMEM <= 227 * 1024, "shared memory");
  static unsigned long long attr_done = 0;
  const auto fn = prompt_attn_kernel<T, DH, NT>;
  if (C::LAUNCH_REGS < 256) {
    // The register split counts on LAUNCH_REGS per thread at launch: with fewer,
    // the softmax warps would wait for theirs without end.  A build that gave the
    // kernel another number is refused
    static int checked = 0;
    if (!__atomic_load_n(&checked, __ATOMIC_ACQUIRE)) {
      cudaFuncAttributes fa;
      if (cudaFuncGetAttributes(&fa, reinterpret_cast<const void*>(fn)) != cudaSuccess) {
        cudaGetLastError();
        return QI_ERR_CUDA;
      }
      if (fa.numRegs != C::LAUNCH_REGS) return QI_ERR_UNSUPPORTED;
      __atomic_store_n(&checked, 1, __ATOMIC_RELEASE);
    }
  }
  if (smem_optin(reinterpret_cast<const void*>(fn), C::SMEM, &attr_done) != QI_OK) return QI_ERR_CUDA;
  const dim3 grid(d.items, d.a.heads / d.P);
  const int st = launch_dependent(fn, grid, C::THREADS, C::SMEM, d, stream);
  if (st != QI_OK || d.splits == 1) return st;
  const PromptAttnArgs& a = d.a;
  // warps per head: several while there are few rows (a row's splits are a chain
  // of loads otherwise), one when the rows alone fill the device
  const long long rows = static_cast<long long>(a.total_q) * a.heads;
  int warps = d.splits >= 16 ? 8 : (d.splits >= 8 ? 4 : (d.splits >= 4 ? 2 : 1));
  while (warps > 1 && rows * warps > 8192) warps /= 2;
  const int per_cta = 8 / warps;
  const JoinDev j{a.out, a.o_row, a.o_head, a.q_begin, a.q_end, d.part, d.ml, d.used, a.batch, a.total_q, a.heads, a.head_dim,
                  warps, d.splits, d.sc};
  return launch_dependent(prompt_attn_join_kernel<T, DH>, dim3(a.total_q, (a.heads + per_cta - 1) / per_cta), 256, 0, j, stream);
}

template <typename T>
int launch_typed(const PromptAttnDev& d, int nt, int dh, cudaStream_t stream) {
  if (dh == 64) return nt == 1 ? launch_tiles<T, 64, 1>(d, stream) : launch_tiles<T, 64, 2>(d, stream);
  return nt == 1 ? launch_tiles<T, 128, 1>(d, stream) : launch_tiles<T, 128, 2>(d, stream);
}

}  // namespace

long long prompt_attention_workspace(int heads, int kv_heads, int head_dim, int batch, int total_q, int max_k) {
  if (batch == 0 || total_q == 0) return 0;
  const Plan p = plan_of(heads, kv_heads, head_dim, batch, total_q, max_k, device_num_sms());
  if (p.splits == 1) return 0;
  return static_cast<long long>(total_q) * heads * (p.splits * (p.dh * 4ll + 8) + 4);
}

int prompt_attention_launch(const PromptAttnArgs& a, cudaStream_t stream) {
  const Plan p = plan_of(a.heads, a.kv_heads, a.head_dim, a.batch, a.total_q, a.max_k, device_num_sms());
  if (p.items > 0x7fffffffll) return QI_ERR_UNSUPPORTED;
  PromptAttnDev d;
  memset(&d, 0, sizeof(d));
  d.a = a;
  d.P = p.P;
  d.T = p.T;
  d.packs = p.packs;
  d.items = static_cast<int>(p.items);
  d.splits = p.splits;
  d.sc = (a.scale < 0.0f ? -a.scale : a.scale) * 1.4426950408889634f;
  // scale 0: the smallest subnormal number.  No finite score makes an exponent
  // past 2^-20 with it (weights 1), and masked scores stay at -inf, where 0 would
  // make them NaN
  constexpr float TINY = 1.40129846e-45f;
  if (d.sc < TINY) d.sc = TINY;
  d.step = fminf(8.0f / d.sc, 3.4028235e38f);
  d.negate = a.scale < 0.0f ? 1u << 13 : 0u;
  if (p.splits > 1) {
    const long long rows = static_cast<long long>(a.total_q) * a.heads;
    d.part = static_cast<float*>(a.workspace);
    d.ml = reinterpret_cast<float2*>(d.part + p.splits * rows * p.dh);
    d.used = reinterpret_cast<int*>(d.ml + p.splits * rows);
  }
  // a dimension of one element has no stride to go by: any valid one will do
  auto stride = [](long long s, long long n) { return static_cast<cuuint64_t>(n > 1 ? s * 2 : 16); };
  const cuuint64_t dim = a.head_dim;
  // Q, out: (d, head of the pack, token, pack): a tile's rows are token-major, heads inside
  auto rows = [&](CUtensorMap* tm, const void* base, long long row, long long head) {
    cuuint64_t dims[4] = {dim, static_cast<cuuint64_t>(p.P), static_cast<cuuint64_t>(a.total_q),
                          static_cast<cuuint64_t>(a.heads / p.P)};
    cuuint64_t str[3] = {stride(head, p.P), stride(row, a.total_q), stride(head * p.P, a.heads / p.P)};
    cuuint32_t box[4] = {64, static_cast<cuuint32_t>(p.P), static_cast<cuuint32_t>(p.T), 1};
    return encode_heads(tm, a.dtype, base, 4, dims, str, box);
  };
  if (rows(&d.tmQ, a.q, a.q_row, a.q_head) != QI_OK || rows(&d.tmO, a.out, a.o_row, a.o_head) != QI_OK) return QI_ERR_CUDA;
  // K, V: (d, kv head, row); without rows the base is never read, and any will do
  auto kv = [&](CUtensorMap* tm, const void* base, long long row, long long head) {
    cuuint64_t dims[3] = {dim, static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.total_k > 0 ? a.total_k : 1)};
    cuuint64_t str[2] = {stride(head, a.kv_heads), stride(row, a.total_k)};
    cuuint32_t box[3] = {64, 1, BKV};
    return encode_heads(tm, a.dtype, a.total_k > 0 ? base : a.q, 3, dims, str, box);
  };
  if (kv(&d.tmK, a.k, a.k_row, a.k_head) != QI_OK || kv(&d.tmV, a.v, a.v_row, a.v_head) != QI_OK) return QI_ERR_CUDA;
  return a.dtype == QI_DT_BF16 ? launch_typed<__nv_bfloat16>(d, p.nt, p.dh, stream)
                               : launch_typed<__half>(d, p.nt, p.dh, stream);
}

int prompt_attention_take_error(int* bad) {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, g_prompt_attn_err, sizeof(int)) != cudaSuccess) return QI_ERR_CUDA;
  if (h) {
    *bad = 1;
    h = 0;
    if (cudaMemcpyToSymbol(g_prompt_attn_err, &h, sizeof(int)) != cudaSuccess) return QI_ERR_CUDA;
  }
  return QI_OK;
}

}  // namespace qi
