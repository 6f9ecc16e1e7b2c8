// The int8 matrix product C = epi(A @ B^T): A [M,K] tokens, B [N,K] channels,
// both running along K, int32 sums (exact up to K = 131071), one fp32 scale per
// token and per channel applied to the finished sum.
//
// k_int8_pair: the tensor-core kernel, persistent over 256 x BN output tiles, one
// tile per pair of CTAs (tcgen05.mma.cta_group::2.kind::i8, 256 x BN x 32). Both
// operands run along k, so a stage is 128 rows of A and BN / 2 rows of B per CTA,
// 128 k values (128 bytes) each, in the 128-byte swizzle. The int32 accumulator
// is double-buffered in TMEM, so that the epilogue of one tile runs beside the
// next tile's products. BN is 256 where the tiles fill the GPU and 128 or 64
// where they do not (pair_plan); a short last wave of long tiles is split along k
// over idle pairs, whose int32 parts are exact in any order.
// k_int8_gemm_any: operands that TMA cannot describe.
#include <atomic>
#include <mutex>

#include "int8_math.cuh"
#include "int8_sched.h"
#include "kernel_config.h"

namespace tfb200 {

namespace {

// Any alignment: 64 x 64 tiles, 64 k values a step in shared memory, dp4a (1024 x 4096 x
// 4096 706 us, 17 in the layout TMA reads).
constexpr int kAnyTile = 64, kAnyK = 64;

__device__ __forceinline__ uint32_t load4(const int8_t* p, int k, int K) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (k + j < K) w |= static_cast<uint32_t>(static_cast<uint8_t>(p[k + j])) << (8 * j);
  return w;
}

__global__ void __launch_bounds__(256) k_int8_gemm_any(const int8_t* A, int64_t lda, const int8_t* B, int64_t ldb,
                                                       const Int8Epi e) {
  __shared__ uint32_t sa[kAnyTile][kAnyK / 4 + 1], sb[kAnyTile][kAnyK / 4 + 1], sums[kAnyTile * kAnyTile];
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kAnyTile;
  const int row = threadIdx.x >> 2, seg = (threadIdx.x & 3) * 4;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t n0 = static_cast<int64_t>(blockIdx.y) * kAnyTile; n0 < e.N;
       n0 += static_cast<int64_t>(gridDim.y) * kAnyTile) {
    int32_t acc[4][4] = {};
    for (int k0 = 0; k0 < e.K; k0 += kAnyK) {
      const bool a_in = m0 + row < e.M, b_in = n0 + row < e.N;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = k0 + (seg + j) * 4;
        sa[row][seg + j] = a_in ? load4(A + (m0 + row) * lda, k, e.K) : 0u;
        sb[row][seg + j] = b_in ? load4(B + (n0 + row) * ldb, k, e.K) : 0u;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kAnyK / 4; ++k) {
        int32_t a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = static_cast<int32_t>(sa[ty + 16 * i][k]);
          b[i] = static_cast<int32_t>(sb[tx + 16 * i][k]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
      }
      __syncthreads();
    }
    // The sums go through shared memory to eight neighbouring columns of a row
    // per thread.
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[(ty + 16 * i) * kAnyTile + tx + 16 * j] = static_cast<uint32_t>(acc[i][j]);
    __syncthreads();
#pragma unroll 1
    for (int it = threadIdx.x; it < kAnyTile * kAnyTile / 8; it += 256) {
      const int64_t m = m0 + it / (kAnyTile / 8);
      const int c = it % (kAnyTile / 8) * 8;
      const int n = static_cast<int>(n0) + c;
      if (m >= e.M || n >= e.N) continue;
      uint32_t v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = sums[it / (kAnyTile / 8) * kAnyTile + c + j];
      float f[8];
      int8_values(e, v, e.a_scale[m], int8_cols(e, n, e.vec_cols), f);
      if (e.residual) int8_residual(e, m, n, e.vec_res, f);
      int8_store(e, m, n, e.vec_out, f);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------ CTA-pair kernel

constexpr int kBM = kPairBM;               // rows of A, and rows of B, per CTA
constexpr int kBK = kPairBK;               // k values per stage (128 bytes)
constexpr uint32_t kABytes = kBM * kBK;    // A's share of a stage: 16 KiB
constexpr int kEpiWarps = cfg::kPairEpiWarps;
constexpr uint32_t kStageOut = 32 * 64;    // one staged block: 32 rows of 64 bytes
constexpr int kGroup = cfg::kGroupM;       // row tiles per raster group
constexpr int kMaxStages = 9;

template <int BN>
struct Geo {
  static constexpr uint32_t kBBytes = BN / 2 * kBK;
  static constexpr int kStages = BN == 256 ? 6 : BN == 128 ? 8 : 9;
  static constexpr int kChunks = BN / 64;  // 32-column chunks per epilogue warp
};

struct PairCtl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  // Scales and bias of the tile's columns, for the epilogue. Read from global
  // memory chunk by chunk they cost an L2 round trip each behind the operands'
  // traffic, longer than the products of a 4096-deep tile.
  alignas(16) float sb[kMaxBN];
  alignas(16) uint16_t bias[kMaxBN];
};

template <int BN>
constexpr size_t pair_smem() {
  return 1024 + Geo<BN>::kStages * (kABytes + Geo<BN>::kBBytes) + static_cast<size_t>(kEpiWarps) * 2 * kStageOut +
         sizeof(PairCtl);
}
static_assert(pair_smem<256>() <= 227 * 1024 && pair_smem<128>() <= 227 * 1024 && pair_smem<64>() <= 227 * 1024,
              "shared memory of one CTA");

struct PairParams {
  Int8Epi e;
  int fast;  // the residual and C are laid out in 16-byte steps; C is stored with TMA
  int b_prefetch, a_early;
  sched::PairSched ps;
  int32_t* slots;
  int* flags;
  int* status;
  uint64_t timeout_ns;
};

__device__ __forceinline__ void tile_of(int t, int num_m, int num_n, int& tm, int& tn) {
  const int per_group = kGroup * num_n;
  const int g = t / per_group;
  const int rows = min(num_m - g * kGroup, kGroup);
  const int local = t - g * per_group;
  tm = g * kGroup + local % rows;
  tn = local / rows;
}

__device__ __forceinline__ void give_up(PairCtl* ctl, int* status) {
  ctl->abort = 1;
  atomicExch(status, kDevTimeout);
}

// 16 bytes at 16-byte unit u of the lane's row in a staged block (64-byte
// swizzle: conflict-free for eight rows).
__device__ __forceinline__ void stage16(uint32_t buf, int lane, int u, uint32_t a, uint32_t b, uint32_t c,
                                        uint32_t d) {
  const uint32_t at = buf + static_cast<uint32_t>(lane * 64 + ((u ^ ((lane >> 1) & 3)) << 4));
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Barrier of the four epilogue warps that share a half of the tile's columns.
__device__ __forceinline__ void half_bar(int half) { asm volatile("bar.sync %0, 128;" ::"r"(half + 1) : "memory"); }

// PLAIN: an fp32 result whose rows lie in 16-byte steps, without a residual, as an
// MLP's hidden block is (the code of the other forms costs registers).
template <bool PLAIN, int BN>
__global__ void __launch_bounds__(cfg::kPairThreads, 1)
    k_int8_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmC, const PairParams p) {
  constexpr int kStages = Geo<BN>::kStages, kChunks = Geo<BN>::kChunks;
  constexpr uint32_t kBBytes = Geo<BN>::kBBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sA = smem;
  uint8_t* sB = sA + kStages * kABytes;
  uint8_t* sC = sB + kStages * kBBytes;
  PairCtl* ctl = reinterpret_cast<PairCtl*>(sC + kEpiWarps * 2 * kStageOut);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&ctl->full[s]), 1);
      mbar_init(smem_u32(&ctl->empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&ctl->tfull[b]), 1);
      mbar_init(smem_u32(&ctl->tempty[b]), 2 * kEpiWarps);  // the epilogue warps of both CTAs
    }
    mbar_init(smem_u32(&ctl->drain), 1);
    ctl->abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (p.fast) tma_prefetch_desc(&tmC);
  }
  if (warp == 2) {
    tmem_alloc_pair(smem_u32(&ctl->tmem_base), 2 * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers exist before any remote arrival
  tc_fence_after();
  const uint32_t tmem_base = ctl->tmem_base;
  grid_dep_launch();
  if (warp != 0) grid_dep_wait();  // the producer waits below, after its weight prefetch

  const int pair = blockIdx.x >> 1;
  const sched::PairSched& ps = p.ps;
  const int nwork = item_count(ps, pair);
  const int num_m = (p.e.M + 2 * kBM - 1) / (2 * kBM);
  const int num_n = (p.e.N + BN - 1) / BN;

  if (warp == 0) {
    // ------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      // The first stages of B, if the preceding kernel does not write it, are
      // requested while that kernel finishes; A follows after the wait, unless
      // that kernel does not write it either.
      int npre = 0;
      if (p.b_prefetch && nwork > 0) {
        const PairWork w = item_at(ps, pair, 0);
        int tm, tn;
        tile_of(w.tile, num_m, num_n, tm, tn);
        npre = min(kStages, w.k1 - w.k0);
        for (int s = 0; s < npre; ++s) {
          const uint32_t fb = mapa_shared(smem_u32(&ctl->full[s]), 0);
          if (leader) mbar_arrive_expect_tx(smem_u32(&ctl->full[s]), 2 * (kABytes + kBBytes));
          tma_load_2d_pair(smem_u32(sB + s * kBBytes), &tmB, fb, (w.k0 + s) * kBK,
                           tn * BN + static_cast<int>(rank) * (BN / 2));
        }
      }
      if (!p.a_early) grid_dep_wait();
      for (int i = 0; i < nwork && ok; ++i) {
        const PairWork w = item_at(ps, pair, i);
        int tm, tn;
        tile_of(w.tile, num_m, num_n, tm, tn);
        for (int kb = w.k0; kb < w.k1; ++kb) {
          const bool pre = i == 0 && kb - w.k0 < npre;  // armed, B in flight
          if (!pre && !mbar_wait(smem_u32(&ctl->empty[stage]), phase ^ 1u, &ctl->abort, p.timeout_ns)) {
            give_up(ctl, p.status);
            ok = false;
            break;
          }
          const uint32_t fb = mapa_shared(smem_u32(&ctl->full[stage]), 0);
          if (leader && !pre) mbar_arrive_expect_tx(smem_u32(&ctl->full[stage]), 2 * (kABytes + kBBytes));
          tma_load_2d_pair(smem_u32(sA + stage * kABytes), &tmA, fb, kb * kBK,
                           tm * 2 * kBM + static_cast<int>(rank) * kBM);
          if (!pre)
            tma_load_2d_pair(smem_u32(sB + stage * kBBytes), &tmB, fb, kb * kBK,
                             tn * BN + static_cast<int>(rank) * (BN / 2));
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        // Copies already issued land within microseconds; give them time before
        // the cluster tears down.
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 1000000ull) {
        }
      }
    }
  } else if (warp == 1) {
    // --------------------------------------------------- MMA issuer (leader)
    if (lane == 0 && leader) {
      constexpr uint32_t idesc = idesc_i8(2 * kBM, BN);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < nwork && ok; ++i) {
        const PairWork w = item_at(ps, pair, i);
        const int acc = i & 1;
        const uint32_t use = static_cast<uint32_t>(i >> 1);
        if (!mbar_wait(smem_u32(&ctl->tempty[acc]), (use & 1u) ^ 1u, &ctl->abort, p.timeout_ns)) {
          give_up(ctl, p.status);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = w.k0; kb < w.k1; ++kb) {
          if (!mbar_wait(smem_u32(&ctl->full[stage]), phase, &ctl->abort, p.timeout_ns)) {
            give_up(ctl, p.status);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + stage * kABytes);
          const uint32_t b0 = smem_u32(sB + stage * kBBytes);
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)
            mma_i8_pair(d, sdesc_sw128(a0 + k * 32, 16, 1024), sdesc_sw128(b0 + k * 32, 16, 1024), idesc,
                        (kb != w.k0 || k != 0) ? 1u : 0u);
          mma_commit_pair_both(smem_u32(&ctl->empty[stage]), 0x3);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) mma_commit_pair_both(smem_u32(&ctl->tfull[acc]), 0x3);
      }
      mma_commit_pair(smem_u32(&ctl->drain));
      const uint64_t t0 = global_ns();
      while (!mbar_test(smem_u32(&ctl->drain), 0) && global_ns() - t0 < p.timeout_ns) {
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------- epilogue (both CTAs)
    // Warp w reads TMEM lane quadrant q = w % 4 (rows q*32 .. q*32+31 of this
    // CTA's 128) and half of the tile's column chunks.
    const int q = warp & 3;
    const int ew = warp - 4;
    const int c0 = (ew >> 2) * kChunks;
    const int r = q * 32 + lane;
    const uint32_t bufs = smem_u32(sC) + static_cast<uint32_t>(ew * 2) * kStageOut;
    // Of 16-bit results, a store's block is staged while the one before it may
    // still be read, so the warp's stores take its two buffers in turn. They are
    // counted over all its tiles: a tile may end after any number of them (one in
    // a 64-column tile, or where the matrix ends).
    uint32_t odd_store = 0;
    for (int i = 0; i < nwork; ++i) {
      const PairWork w = item_at(ps, pair, i);
      int tm, tn;
      tile_of(w.tile, num_m, num_n, tm, tn);
      const int acc = i & 1;
      const uint32_t use = static_cast<uint32_t>(i >> 1);
      const int64_t row0 = static_cast<int64_t>(tm) * 2 * kBM + static_cast<int64_t>(rank) * kBM + q * 32;
      const int64_t row = row0 + lane;
      const bool row_in = row < p.e.M;
      const bool part = w.role == sched::kPart, fix = w.role == sched::kMain;
      // While the tile's products run: the row's scale, a column's scale and bias
      // per thread (four warps share a half of the columns), the residual into L2.
      float sa = 0.0f;
      if (!part) {
        const int n = tn * BN + c0 * 32 + r;
        const bool col_in = r < BN / 2 && n < p.e.N;
        const float sb = col_in ? p.e.b_scale[n] : 0.0f;
        const uint16_t bias = p.e.bias && col_in ? reinterpret_cast<const uint16_t*>(p.e.bias)[n] : uint16_t(0);
        if (row_in) {
          sa = p.e.a_scale[row];
          if (!PLAIN && p.e.residual)
            for (int c = c0; c < c0 + kChunks && tn * BN + c * 32 < p.e.N; c += 2)
              prefetch_l2(p.e.residual + row * p.e.ldr + tn * BN + c * 32);
        }
        half_bar(ew >> 2);  // the half's warps are done with the last tile's columns
        if (r < BN / 2) {
          ctl->sb[c0 * 32 + r] = sb;
          ctl->bias[c0 * 32 + r] = bias;
        }
        half_bar(ew >> 2);
      }
      bool ok = mbar_wait(smem_u32(&ctl->tfull[acc]), use & 1u, &ctl->abort, p.timeout_ns);
      ok = __all_sync(0xffffffffu, ok);
      // A warp whose wait ran out goes on through the items, so that the other
      // warps of its half meet it at their barriers; their waits end at once.
      if (!ok) {
        if (lane == 0) give_up(ctl, p.status);
        continue;
      }
      tc_fence_after();
      const uint32_t tacc = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(acc * BN);
      // A split tile's flags: one per part and epilogue warp.
      int* const flag = p.flags + (w.slot * 2 + static_cast<int>(rank)) * kEpiWarps + ew;
      if (fix && row0 < p.e.M) {
        // Lane j waits for part j (acquire); the warp's barrier passes that on.
        if (lane < ps.parts) {
          const uint64_t t0 = global_ns();
          while (ok && ld_acquire_gpu(flag + lane * 2 * kEpiWarps) == 0)
            if (ctl->abort || global_ns() - t0 > p.timeout_ns) ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (lane == 0) give_up(ctl, p.status);
          continue;
        }
      }
      for (int c = c0; c < c0 + kChunks; ++c) {
        const int col0 = tn * BN + c * 32;
        if (col0 >= p.e.N || row0 >= p.e.M) break;  // warp-uniform: nothing of this block is in the matrix
        // Slots: [chunk][column / 4][row][4], so that a warp's 16-byte accesses
        // cover 512 contiguous bytes.
        int4* slot = reinterpret_cast<int4*>(p.slots + (static_cast<int64_t>(w.slot) * 2 + rank) * (kBM * BN)) +
                     c * 8 * kBM + r;
        uint4 res[4];
        const bool whole = col0 + 32 <= p.e.N;
        if (!PLAIN && p.fast && p.e.residual && whole && row_in && !part) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            res[u] = *reinterpret_cast<const uint4*>(p.e.residual + row * p.e.ldr + col0 + u * 8);
        }
        uint32_t v[32];
        tmem_ld_32cols(tacc + static_cast<uint32_t>(c * 32), v);
        tmem_wait_ld();
        if (part) {
          // A helper's rows of the chunk go to its slot.
#pragma unroll
          for (int k = 0; k < 8; ++k)
            __stcg(slot + k * kBM, make_int4(static_cast<int>(v[4 * k]), static_cast<int>(v[4 * k + 1]),
                                             static_cast<int>(v[4 * k + 2]), static_cast<int>(v[4 * k + 3])));
          continue;
        }
        if (fix) {
#pragma unroll 2
          for (int j = 0; j < ps.parts; ++j) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int4 add = __ldcg(slot + j * (kBM * BN / 2) + k * kBM);
              v[4 * k] += static_cast<uint32_t>(add.x);
              v[4 * k + 1] += static_cast<uint32_t>(add.y);
              v[4 * k + 2] += static_cast<uint32_t>(add.z);
              v[4 * k + 3] += static_cast<uint32_t>(add.w);
            }
          }
        }
        const bool f32 = PLAIN || p.e.out == kInt8OutF32;
        const uint32_t buf = bufs + (f32 ? 0u : odd_store * kStageOut);
        uint64_t v2[16];  // fp32 pairs
        {
          const ulonglong2* sb = reinterpret_cast<const ulonglong2*>(ctl->sb + c * 32);
          const uint4* bias = reinterpret_cast<const uint4*>(ctl->bias + c * 32);
          const uint64_t sa2 = f2(sa, sa);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const ulonglong2 s0 = sb[2 * u], s1 = sb[2 * u + 1];
            const uint4 b = bias[u];
            const uint64_t s4[4] = {s0.x, s0.y, s1.x, s1.y};
            const uint32_t b4[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              v2[u * 4 + j] =
                  int8_scaled(v[u * 8 + 2 * j], v[u * 8 + 2 * j + 1], sa2, s4[j], f2_from_bf16x2(b4[j]));
          }
        }
        if (p.e.gelu == kGeluErf) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v2[j] = int8_gelu_erf(v2[j]);
        } else if (p.e.gelu == kGeluTanh) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v2[j] = int8_gelu_tanh(v2[j]);
        }
        float f[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) f2_split(v2[j], f[2 * j], f[2 * j + 1]);
        if (!PLAIN && !p.fast) {
          // The residual or C is not laid out in 16-byte steps: the block goes
          // through shared memory (as fp32 in both buffers, unit j ^ row of a row)
          // and is finished row by row, a lane per column.
#pragma unroll
          for (int j = 0; j < 32; ++j)
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(bufs + static_cast<uint32_t>((lane * 32 + (j ^ lane)) * 4)),
                         "f"(f[j])
                         : "memory");
          __syncwarp();
          const int n = col0 + lane;
          const int rows = n < p.e.N ? static_cast<int>(min(static_cast<int64_t>(32), p.e.M - row0)) : 0;
#pragma unroll 1
          for (int k0 = 0; k0 < rows; k0 += 8) {
            float x[8], y[8] = {};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              asm volatile("ld.shared.b32 %0, [%1];"
                           : "=f"(x[k])
                           : "r"(bufs + static_cast<uint32_t>(((k0 + k) * 32 + (lane ^ (k0 + k))) * 4))
                           : "memory");
              if (p.e.residual && k0 + k < rows) y[k] = __bfloat162float(p.e.residual[(row0 + k0 + k) * p.e.ldr + n]);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              if (k0 + k >= rows) break;
              const int64_t at = (row0 + k0 + k) * p.e.ldc + n;
              const float z = __fadd_rn(x[k], y[k]);
              if (f32)
                static_cast<float*>(p.e.C)[at] = z;
              else
                static_cast<bf16*>(p.e.C)[at] = __float2bfloat16_rn(z);
            }
          }
          __syncwarp();
          continue;
        }
        if (!PLAIN && p.e.residual && row_in) {
          if (whole) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const uint32_t r8[4] = {res[u].x, res[u].y, res[u].z, res[u].w};
#pragma unroll
              for (int j = 0; j < 8; ++j)
                f[u * 8 + j] = __fadd_rn(f[u * 8 + j], (j & 1) ? bf16_hi(r8[j >> 1]) : bf16_lo(r8[j >> 1]));
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col0 + j < p.e.N)
                f[j] = __fadd_rn(f[j], __bfloat162float(p.e.residual[row * p.e.ldr + col0 + j]));
          }
        }
        // The store that used this buffer has read it: 16-bit results, all but the
        // last (which used the other); fp32 results fill both, so all of them.
        if (lane == 0) {
          if (f32)
            bulk_wait_read<0>();
          else
            bulk_wait_read<1>();
        }
        __syncwarp();
        if (f32) {
          // Two blocks of 32 x 16 fp32 values.
#pragma unroll
          for (int u = 0; u < 8; ++u)
            stage16(buf + static_cast<uint32_t>(u >> 2) * kStageOut, lane, u & 3, __float_as_uint(f[4 * u]),
                    __float_as_uint(f[4 * u + 1]), __float_as_uint(f[4 * u + 2]), __float_as_uint(f[4 * u + 3]));
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            stage16(buf, lane, u, pack_bf16(f[u * 8], f[u * 8 + 1]), pack_bf16(f[u * 8 + 2], f[u * 8 + 3]),
                    pack_bf16(f[u * 8 + 4], f[u * 8 + 5]), pack_bf16(f[u * 8 + 6], f[u * 8 + 7]));
        }
        // Rows and columns past the matrix are clipped.
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tmC, buf, col0, static_cast<int32_t>(row0));
          if (f32 && col0 + 16 < p.e.N)
            tma_store_2d(&tmC, buf + kStageOut, col0 + 16, static_cast<int32_t>(row0));
          bulk_commit();
        }
        odd_store ^= 1u;
      }
      if (part) {
        // One release for the warp's rows (one per chunk cost 1.3 us each).
        __syncwarp();
        if (lane == 0) st_release_gpu(flag, 1);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        const uint32_t te = smem_u32(&ctl->tempty[acc]);
        if (leader)
          mbar_arrive(te);
        else
          mbar_arrive_cluster(mapa_shared(te, 0));
      }
    }
    if (lane == 0 && (PLAIN || p.fast)) bulk_wait_all();  // staged stores have left shared memory
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still touch its barriers or shared memory
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * BN);
  }
}

bool al(const void* p, unsigned b) { return (reinterpret_cast<uintptr_t>(p) & (b - 1)) == 0; }

using PairKernel = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const PairParams);
template <int BN>
PairKernel pair_kernel(bool plain) {
  return plain ? k_int8_pair<true, BN> : k_int8_pair<false, BN>;
}
PairKernel pair_kernel(bool plain, int bn) {
  return bn == 256 ? pair_kernel<256>(plain) : bn == 128 ? pair_kernel<128>(plain) : pair_kernel<64>(plain);
}
size_t pair_smem(int bn) { return bn == 256 ? pair_smem<256>() : bn == 128 ? pair_smem<128>() : pair_smem<64>(); }

// Per-device set-up of the first call; calls may come from several host
// threads. *pairs: how many pairs are resident at once.
cudaError_t pair_ready(int* pairs) {
  static std::mutex mu;
  static std::atomic<int> resident[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  *pairs = resident[dev].load(std::memory_order_acquire);
  if (*pairs > 0) return cudaSuccess;
  std::lock_guard<std::mutex> lock(mu);
  for (const int bn : {64, 128, 256})
    for (const bool plain : {false, true}) {
      e = cudaFuncSetAttribute(pair_kernel(plain, bn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(pair_smem(bn)));
      if (e != cudaSuccess) return e;
    }
  cudaLaunchConfig_t q{};
  q.gridDim = dim3(static_cast<unsigned>(sm_count()), 1, 1);
  q.blockDim = dim3(cfg::kPairThreads, 1, 1);
  q.dynamicSmemBytes = pair_smem(kMaxBN);  // one CTA per SM in every form
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim = {2, 1, 1};
  q.attrs = a;
  q.numAttrs = 1;
  int n = 0;
  e = cudaOccupancyMaxActiveClusters(&n, pair_kernel(false, kMaxBN), &q);
  if (e == cudaSuccess && n <= 0) e = cudaErrorLaunchOutOfResources;
  if (e != cudaSuccess) return e;
  resident[dev].store(n, std::memory_order_release);
  *pairs = n;
  return cudaSuccess;
}

int launch_pair(const Int8Gemm& g, cudaStream_t s, std::string* err) {
  int resident = 0;
  cudaError_t e = pair_ready(&resident);
  if (e != cudaSuccess) {
    *err = std::string("int8 pair gemm set-up: ") + cudaGetErrorString(e);
    return -3;
  }
  PairParams p{};
  p.e = int8_epi(g);
  p.status = device_status_ptr(err);
  if (!p.status) return -3;
  p.timeout_ns = wait_limit_ns();
  const int esz = g.out == kInt8OutF32 ? 4 : 2;
  p.fast = al(g.C, 16) && g.ldc * esz % 16 == 0 && (!g.residual || p.e.vec_res);
  p.b_prefetch = g.b_stable;
  p.a_early = g.a_stable;
  const PairPlan plan = pair_plan(g.M, g.N, g.K);
  CUtensorMap ta{}, tb{}, tc{};
  if (!int8_map(&ta, g.A, g.M, g.K, g.lda, kBM, err) ||
      !int8_map(&tb, g.B, g.N, g.K, g.ldb, static_cast<uint32_t>(plan.bn / 2), err))
    return -3;
  if (p.fast && !make_map_box(&tc, g.C, g.M, g.N, g.ldc, static_cast<uint32_t>(64 / esz), 32,
                                   CU_TENSOR_MAP_SWIZZLE_64B, err,
                                   g.out == kInt8OutF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                   esz))
    return -3;
  p.ps = plan.s;
  if (p.ps.rem > 0 && resident >= kSmPairs) {
    p.flags = static_cast<int*>(g.ws);
    const size_t clear = int8_gemm_ws(g.M, g.N, g.K).clear_bytes;
    p.slots = reinterpret_cast<int32_t*>(static_cast<char*>(g.ws) + clear);
  } else {
    p.ps = sched::plan(p.ps.tiles, p.ps.kblocks, p.ps.tiles < resident ? p.ps.tiles : resident, 0);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * p.ps.pairs), 1, 1);
  cfg.blockDim = dim3(cfg::kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = pair_smem(plan.bn);
  cfg.stream = s;
  cudaLaunchAttribute a[2];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim = {2, 1, 1};
  a[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = a;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, pair_kernel(g.out == kInt8OutF32 && p.fast && !g.residual, plan.bn), ta, tb, tc, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    *err = std::string("int8 pair gemm launch: ") + cudaGetErrorString(e);
    return -3;
  }
  count_launch();
  return 0;
}

}  // namespace

bool int8_map(CUtensorMap* m, const int8_t* base, int64_t rows, int64_t cols, int64_t ld, uint32_t box_rows,
              std::string* err) {
  return make_map_box(m, base, rows, cols, rows > 1 ? ld : (cols + 15) / 16 * 16, kBK, box_rows,
                      CU_TENSOR_MAP_SWIZZLE_128B, err, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1);
}

// The kernel of a product whose operands are aligned, by estimates in us:
//   stream  up to 128 rows: 5.6 + 0.075 per row (slots, arrivals, finish) + weights
//           at 6 TB/s
//   gemv    up to 32 rows: int8_gemv_us
//   pair    2.5 + 0.29 per k-block of its plan + weights at 12 TB/s
// Measured, us, gemv / stream / pair: 1 x 1024 x 1024 2.0 / 6.3 / 5.5, 1 x 4096 x 4096
// 4.4 / 9.7 / 14.3, 8 x 4096 x 16384 13.0 / 16.7, 8 x 8192 x 28672 39.9 / 42.5,
// 16 x 4096 x 4096 5.9 / 10.2, 16 x 8192 x 28672 47.0 / 42.9, 32 x 2048 x 2048 4.8 / 8.8 /
// 7.8, 32 x 4096 x 4096 8.6 / 11.3 / 13.4, 32 x 4096 x 6144 13.6 / 13.1, 64 x 2048 x 2048
// (four tiles of tokens) 11.3 / - / 7.9, 128 x 1024 x 1024 - / 16.1 / 5.8,
// 128 x 4096 x 4096 - / 15.7 / 13.6, 128 x 16384 x 4096 - / 23.3 / 30.8,
// 128 x 8192 x 28672 - / 50.0 / 53.4.
enum Kernel { kPair, kStream, kGemv };
static Kernel kernel_of(int64_t m, int64_t n, int64_t k) {
  if (m > kInt8StreamRows) return kPair;
  const double mb = static_cast<double>(n) * static_cast<double>(k) * 1e-6;
  const double stream = 5.6 + 0.075 * static_cast<double>(m) + mb / 6.0;
  const double pair = 2.5 + 0.29 * pair_plan(m, n, k).cost + mb / 12.0;
  if (m <= kInt8GemvRows && int8_gemv_us(m, n, k) <= (stream < pair ? stream : pair)) return kGemv;
  return stream <= pair ? kStream : kPair;
}

Int8GemmWs int8_gemm_ws(int64_t m, int64_t n, int64_t k) {
  Int8GemmWs w;
  if (k <= 0 || pair_tiles(m, n, kMaxBN) > (1 << 30)) return w;
  const Kernel kernel = kernel_of(m, n, k);
  if (kernel == kGemv) return w;
  if (kernel == kStream) return int8_stream_ws(m, n);
  const sched::PairSched ps = pair_plan(m, n, k).s;
  if (ps.rem > 0) {
    w.clear_bytes = (static_cast<size_t>(ps.rem) * ps.parts * 2 * kEpiWarps * sizeof(int) + 255) / 256 * 256;
    w.total = w.clear_bytes + static_cast<size_t>(ps.rem) * ps.parts * sched::kSlotBytes;
  }
  return w;
}

int run_int8_gemm(const Int8Gemm& g, cudaStream_t stream, std::string* err) {
  if (g.M > (int64_t(1) << 30) || g.N > (int64_t(1) << 30) || g.K > kInt8MaxK) {
    *err = "dimension too large";
    return -2;
  }
  // TMA describes operands that start on 16-byte boundaries with row strides
  // that are multiples of 16 bytes (one row has no stride).
  if (g.K > 0 && al(g.A, 16) && al(g.B, 16) && (g.lda % 16 == 0 || g.M == 1) && (g.ldb % 16 == 0 || g.N == 1) &&
      pair_tiles(g.M, g.N, kMaxBN) <= (1 << 30))
    switch (kernel_of(g.M, g.N, g.K)) {
      case kGemv: return run_int8_gemv(g, stream, err);
      case kStream: return run_int8_stream(g, stream, err);
      case kPair: return launch_pair(g, stream, err);
    }
  const int64_t by = (g.N + kAnyTile - 1) / kAnyTile;
  const dim3 grid(static_cast<unsigned>((g.M + kAnyTile - 1) / kAnyTile),
                  static_cast<unsigned>(by < 65535 ? by : 65535));
  k_int8_gemm_any<<<grid, 256, 0, stream>>>(g.A, g.lda, g.B, g.ldb, int8_epi(g));
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    *err = std::string("int8 gemm launch: ") + cudaGetErrorString(e);
    return -3;
  }
  count_launch();
  return 0;
}

}  // namespace tfb200
