// The int8 product for few rows: HBM-bound, so its work is to stream B (the
// weights) at full bandwidth from every SM.
//
// The product is formed transposed, acc^T = B A^T: the MMA's M side is 128
// channels (rows of B) and its N side the tokens, rounded up to 16. Work units
// are blocks of 128 channels x 128 k values (16 KiB of B); the units, channel
// block by channel block, are cut into gridDim.x contiguous ranges of equal
// length, so every SM streams the same number of bytes. A CTA sums the part of
// each channel block that lies in its range in TMEM. A block that lies whole in
// one range is finished by its CTA; otherwise each CTA writes its int32 sums to
// its slot (block + CTA, unique because the ranges are contiguous), and the last
// to arrive (a counter) adds the slots and finishes the block. int32 sums are
// exact in any order, so equal calls give equal bits.
//
// Only the counters must be zero on entry; the launch before clears them. The
// first ring of B is requested before that launch has completed (it does not
// write B), with an evict-first policy so that the stream does not push slots
// and activations out of L2; A follows after the wait.
//
// Warps: 0 TMA producer, 1 MMA issuer, 2 TMEM allocator, 4-11 epilogue. All
// waits are bounded (kDevTimeout in the status word).
#include <atomic>
#include <mutex>

#include "int8_math.cuh"
#include "kernel_config.h"

namespace tfb200 {

namespace {

constexpr int kN = 128;                 // channels per unit
constexpr int kK = 128;                 // k values per unit
constexpr uint32_t kUnit = kN * kK;     // bytes of B per unit
constexpr int kMaxStages = 12;
constexpr int kBudget = 208 * 1024;     // shared memory of the ring
constexpr int kAcc = 4;                 // TMEM accumulators in rotation
constexpr int kMaxGrid = 160;
constexpr int kEpiThreads = 256;        // warps 4-11, two per TMEM lane quadrant
constexpr int kThreads = 128 + kEpiThreads;

struct Ctl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tfull[kAcc];
  uint64_t tempty[kAcc];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int last;
};

struct StreamParams {
  Int8Epi e;
  int mpad, kblocks, units, stages;
  uint32_t acc_cols, tmem_cols;
  int32_t* slots;
  int* counters;
  int b_prefetch, a_early;
  int pf_units, pf_kblocks, pf_total, pf_grid;  // L2 prefetch of the next product's B
  int* status;
  uint64_t timeout_ns;
};

__device__ __forceinline__ int64_t unit_start(int c, int units, int grid) {
  return static_cast<int64_t>(c) * units / grid;
}
__device__ __forceinline__ int64_t unit_start(int c, int units) {
  return unit_start(c, units, static_cast<int>(gridDim.x));
}
// The CTA whose range holds unit u.
__device__ __forceinline__ int cta_of(int64_t u, int units) {
  const int grid = static_cast<int>(gridDim.x);
  return static_cast<int>(((u + 1) * grid + units - 1) / units - 1);
}

__device__ __forceinline__ void give_up(Ctl* ctl, int* status) {
  ctl->abort = 1;
  atomicExch(status, kDevTimeout);
}

__device__ __forceinline__ void epi_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// AND of `ok` over the epilogue threads, so that all take the same branch.
__device__ __forceinline__ bool epi_all(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(ok ? 1u : 0u)
      : "memory");
  return r != 0;
}

// The epilogue threads run one CTA's segments: slot writes (a lane per channel),
// arrivals, and the finish of completed blocks (a thread per token and eight
// neighbouring channels).
__device__ __forceinline__ void epilogue(const StreamParams& p, Ctl* ctl, const float* s_scale, uint32_t tmem_base) {
  const Int8Epi& e = p.e;
  const int et = threadIdx.x - 128;
  const int q = (et >> 5) & 3, half = et >> 7;
  const int c8 = (et & 15) * 8;  // first of the thread's channels within a block
  const int64_t slot_elems = static_cast<int64_t>(e.M) * kN;
  const int64_t u0 = unit_start(blockIdx.x, p.units), u1 = unit_start(blockIdx.x + 1, p.units);
  int seg = 0;
  for (int nb = static_cast<int>(u0 / p.kblocks); static_cast<int64_t>(nb) * p.kblocks < u1; ++nb, ++seg) {
    const int acc_i = seg % kAcc;
    const int n = nb * kN + c8;
    // What the finish reads besides the sums, requested while the products run
    // (at finishing time these loads wait behind the weight stream).
    const Cols8 cols = int8_cols(e, n, e.vec_cols);
    if (e.residual && n < e.N)
      for (int m = et >> 4; m < e.M; m += kEpiThreads / 16) prefetch_l2(e.residual + m * e.ldr + n);
    const uint32_t parity = static_cast<uint32_t>(seg / kAcc) & 1u;
    if (!epi_all(mbar_wait(smem_u32(&ctl->tfull[acc_i]), parity, &ctl->abort, p.timeout_ns))) {
      if (et == 0) give_up(ctl, p.status);
      return;
    }
    tc_fence_after();
    int32_t* slot = p.slots + (static_cast<int64_t>(nb) + blockIdx.x) * slot_elems + (q * 32 + (et & 31));
#pragma unroll 1
    for (int m = half * 8; m < e.M; m += 16) {
      uint32_t v[8];
      tmem_ld_8cols(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc_i * p.acc_cols + m, v);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (m + j < e.M) __stcg(slot + (m + j) * kN, static_cast<int32_t>(v[j]));
    }
    tc_fence_before();
    mbar_arrive(smem_u32(&ctl->tempty[acc_i]));
    const int64_t first = static_cast<int64_t>(nb) * p.kblocks;
    const int c_first = cta_of(first, p.units), c_last = cta_of(first + p.kblocks - 1, p.units);
    // One thread arrives for the CTA after a barrier (release: its slot before
    // the arrival; acquire: every slot before the reads). A block of this CTA
    // alone needs only the barrier.
    epi_bar();
    if (c_first != c_last) {
      if (et == 0) ctl->last = atom_add_acq_rel_gpu(p.counters + nb, 1) == c_last - c_first;
      epi_bar();
      if (!ctl->last) continue;
    }
    const int32_t* s0 = p.slots + (static_cast<int64_t>(nb) + c_first) * slot_elems + c8;
#pragma unroll 1
    for (int m = et / (kN / 8); n < e.N && m < e.M; m += kEpiThreads / (kN / 8)) {
      uint32_t v[8] = {};
#pragma unroll 4
      for (int c = 0; c <= c_last - c_first; ++c) {
        const int4* s = reinterpret_cast<const int4*>(s0 + c * slot_elems + m * kN);
        const int4 a = __ldcg(s), b = __ldcg(s + 1);
        v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
        v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
      }
      float f[8];
      int8_values(e, v, s_scale[m], cols, f);
      if (e.residual) int8_residual(e, m, n, e.vec_res, f);
      int8_store(e, m, n, e.vec_out, f);
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    k_int8_stream(const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmA,
                  const __grid_constant__ CUtensorMap tmNext, const StreamParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t a_bytes = static_cast<uint32_t>(p.mpad) * kK;
  uint8_t* sB = smem;
  uint8_t* sA = smem + p.stages * kUnit;
  Ctl* ctl = reinterpret_cast<Ctl*>(sA + p.stages * a_bytes);
  float* s_scale = reinterpret_cast<float*>(ctl + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&ctl->full[s]), 1);
      mbar_init(smem_u32(&ctl->empty[s]), 1);
    }
    for (int b = 0; b < kAcc; ++b) {
      mbar_init(smem_u32(&ctl->tfull[b]), 1);
      mbar_init(smem_u32(&ctl->tempty[b]), kEpiThreads);
    }
    mbar_init(smem_u32(&ctl->drain), 1);
    ctl->abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmA);
    if (p.pf_units > 0) tma_prefetch_desc(&tmNext);
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(&ctl->tmem_base), p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctl->tmem_base;
  grid_dep_launch();

  const int64_t u0 = unit_start(blockIdx.x, p.units), u1 = unit_start(blockIdx.x + 1, p.units);
  if (warp == 0) {
    if (lane == 0) {
      const uint64_t evict_first = l2_policy_evict_first();
      int stage = 0, nb = static_cast<int>(u0 / p.kblocks), kb = static_cast<int>(u0 % p.kblocks);
      uint32_t phase = 0, armed = 0, armed_phase = 0;
      bool ok = true;
      // The first ring of B, then its tokens once the preceding grid is done.
      const int pre = p.b_prefetch ? static_cast<int>(min(u1 - u0, static_cast<int64_t>(p.stages))) : 0;
      for (int s = 0; s < pre; ++s) {
        const int64_t u = u0 + s;
        mbar_arrive_expect_tx(smem_u32(&ctl->full[s]), kUnit + a_bytes);
        tma_load_2d_hint(smem_u32(sB + s * kUnit), &tmB, smem_u32(&ctl->full[s]),
                         static_cast<int>(u % p.kblocks) * kK, static_cast<int>(u / p.kblocks) * kN, evict_first);
      }
      if (!p.a_early) grid_dep_wait();
      for (int64_t u = u0; u < u1; ++u) {
        const uint32_t fb = smem_u32(&ctl->full[stage]);
        if (u - u0 >= pre) {
          if (!mbar_wait(smem_u32(&ctl->empty[stage]), phase ^ 1u, &ctl->abort, p.timeout_ns)) {
            give_up(ctl, p.status);
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(fb, kUnit + a_bytes);
          tma_load_2d_hint(smem_u32(sB + stage * kUnit), &tmB, fb, kb * kK, nb * kN, evict_first);
        }
        tma_load_2d(smem_u32(sA + stage * a_bytes), &tmA, fb, kb * kK, 0);
        armed |= 1u << stage;
        armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
        if (++kb == p.kblocks) {
          kb = 0;
          ++nb;
        }
      }
      if (ok && p.pf_units > 0) {
        // This CTA's share of the first units of the next product's ranges. The
        // divisions stay out of the inner loop: the thread holds up the CTA's exit.
        const int all = p.pf_units * p.pf_grid;
        int i = static_cast<int>(unit_start(blockIdx.x, all));
        const int i1 = static_cast<int>(unit_start(blockIdx.x + 1, all));
        while (i < i1) {
          const int c = i / p.pf_units, end = min(i1, (c + 1) * p.pf_units);
          const int first = static_cast<int>(unit_start(c, p.pf_total, p.pf_grid));
          const int last = static_cast<int>(unit_start(c + 1, p.pf_total, p.pf_grid));
          const int u = first + (i - c * p.pf_units);
          int kn = u % p.pf_kblocks, nn = u / p.pf_kblocks;
          for (int n = min(last - u, end - i); n > 0; --n) {
            tma_prefetch_l2_2d(&tmNext, kn * kK, nn * kN);
            if (++kn == p.pf_kblocks) {
              kn = 0;
              ++nn;
            }
          }
          i = end;
        }
      }
      if (!ok) {
        // Let the copies already issued land before shared memory goes away.
        for (int s = 0; s < p.stages; ++s)
          if (armed & (1u << s)) {
            const uint64_t t0 = global_ns();
            while (!mbar_test(smem_u32(&ctl->full[s]), (armed_phase >> s) & 1u) && global_ns() - t0 < p.timeout_ns) {
            }
          }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_i8(kN, p.mpad);
      int stage = 0, seg = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int64_t u = u0; u < u1 && ok; ++seg) {
        const int64_t end = min(u1, (u / p.kblocks + 1) * p.kblocks);
        const int acc_i = seg % kAcc;
        const uint32_t parity = (static_cast<uint32_t>(seg / kAcc) & 1u) ^ 1u;
        if (!mbar_wait(smem_u32(&ctl->tempty[acc_i]), parity, &ctl->abort, p.timeout_ns)) {
          give_up(ctl, p.status);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + acc_i * p.acc_cols;
        for (bool first = true; u < end; ++u, first = false) {
          if (!mbar_wait(smem_u32(&ctl->full[stage]), phase, &ctl->abort, p.timeout_ns)) {
            give_up(ctl, p.status);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t b0 = smem_u32(sB + stage * kUnit), a0 = smem_u32(sA + stage * a_bytes);
#pragma unroll
          for (int k = 0; k < kK / 32; ++k)
            mma_i8(d, sdesc_sw128(b0 + k * 32, 16, 1024), sdesc_sw128(a0 + k * 32, 16, 1024), idesc,
                   first && k == 0 ? 0u : 1u);
          mma_commit(smem_u32(&ctl->empty[stage]));
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) mma_commit(smem_u32(&ctl->tfull[acc_i]));
      }
      mma_commit(smem_u32(&ctl->drain));
      const uint64_t t0 = global_ns();
      while (!mbar_test(smem_u32(&ctl->drain), 0) && global_ns() - t0 < p.timeout_ns) {
      }
    }
  } else if (warp >= 4) {
    grid_dep_wait();  // scales, counters and the residual come from the preceding grids
    for (int m = threadIdx.x - 128; m < p.e.M; m += kEpiThreads) s_scale[m] = p.e.a_scale[m];
    epi_bar();
    epilogue(p, ctl, s_scale, tmem_base);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, p.tmem_cols);
  }
}

// Per-device set-up of the first call; calls may come from several host threads.
cudaError_t ready() {
  static std::mutex mu;
  static std::atomic<bool> done[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  std::lock_guard<std::mutex> lock(mu);
  e = cudaFuncSetAttribute(k_int8_stream, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e != cudaSuccess) return e;
  done[dev].store(true, std::memory_order_release);
  return cudaSuccess;
}

int64_t units_of(int64_t n, int64_t k) { return (n + kN - 1) / kN * ((k + kK - 1) / kK); }

// CTAs of a product: one per SM, or up to a seventh fewer (a quarter over 64 rows,
// where slots weigh more) when that makes every CTA's range end on a channel
// block's border or cut it into equal parts, which spares slots, arrivals and
// finishes. 148 CTAs against fewer, us: 1 x 4096 x 4096 11.0 / 128 CTAs 9.7;
// 16 x 4096 x 6144 13.4 / 144 CTAs 12.3; 128 x 8192 x 28672 53.7 / 112 CTAs 49.7;
// 32 x 8192 x 28672 43.9 / 112 CTAs 44.9; with 96 CTAs the stream itself slows
// down. A block is cut into 8 ranges at most (16 up to 16 rows), because its
// finisher reads them all (at most 8 / all CTAs, us: 32 x 16384 x 96 13.4 / 37.6,
// 128 x 8192 x 1024 18.8 / 29.8, 32 x 16384 x 2048 15.2 / 16.3; 1 x 16384 x 96 with
// at most 16 / 8 / all 10.0 / 11.6 / 16.7).
int grid_of(int64_t m, int64_t n, int64_t k) {
  const int64_t blocks = (n + kN - 1) / kN, units = units_of(n, k);
  const int64_t sms = sm_count() < kMaxGrid ? sm_count() : kMaxGrid, cuts = blocks * (m <= 16 ? 16 : 8);
  const int most = static_cast<int>(sms < cuts ? sms : cuts);
  if (units <= most) return static_cast<int>(units);
  for (int g = most; g >= most - most / (m <= 64 ? 7 : 4); --g)
    if (blocks % g == 0 || g % blocks == 0) return g;
  return most;
}

// Units of the next product's B that are brought into L2 at the end: 78 MB.
constexpr int kPrefetchUnits = 4736;

}  // namespace

Int8GemmWs int8_stream_ws(int64_t m, int64_t n) {
  const int64_t blocks = (n + kN - 1) / kN;
  Int8GemmWs w;
  w.clear_bytes = (static_cast<size_t>(blocks) * sizeof(int) + 255) / 256 * 256;
  w.total = w.clear_bytes + static_cast<size_t>(blocks + kMaxGrid - 1) * static_cast<size_t>(m) * kN * sizeof(int32_t);
  return w;
}

int run_int8_stream(const Int8Gemm& g, cudaStream_t stream, std::string* err) {
  cudaError_t e = ready();
  if (e != cudaSuccess) {
    *err = std::string("int8 stream set-up: ") + cudaGetErrorString(e);
    return -3;
  }
  StreamParams p{};
  p.e = int8_epi(g);
  p.status = device_status_ptr(err);
  if (!p.status) return -3;
  p.timeout_ns = wait_limit_ns();
  p.mpad = static_cast<int>((g.M + 15) / 16 * 16);
  p.kblocks = static_cast<int>((g.K + kK - 1) / kK);
  const int64_t units = units_of(g.N, g.K);
  if (units > (int64_t(1) << 30)) {
    *err = "dimension too large";
    return -2;
  }
  p.units = static_cast<int>(units);
  const uint32_t a_bytes = static_cast<uint32_t>(p.mpad) * kK;
  const int fit = static_cast<int>(kBudget / (kUnit + a_bytes));
  p.stages = fit < kMaxStages ? fit : kMaxStages;
  p.acc_cols = static_cast<uint32_t>(p.mpad <= 32 ? 32 : p.mpad <= 64 ? 64 : 128);
  p.tmem_cols = kAcc * p.acc_cols;
  p.counters = static_cast<int*>(g.ws);
  p.slots = reinterpret_cast<int32_t*>(static_cast<char*>(g.ws) + int8_stream_ws(g.M, g.N).clear_bytes);
  p.b_prefetch = g.b_stable;
  p.a_early = g.a_stable;
  const int grid = grid_of(g.M, g.N, g.K);
  CUtensorMap tb{}, ta{}, tn{};
  if (!int8_map(&tb, g.B, g.N, g.K, g.ldb, kN, err) ||
      !int8_map(&ta, g.A, g.M, g.K, g.lda, static_cast<uint32_t>(p.mpad), err))
    return -3;
  const int64_t next = g.next_b ? units_of(g.next_n, g.next_k) : 0;
  if (next > 0 && next <= (int64_t(1) << 30) && g.next_ld % 16 == 0 &&
      (reinterpret_cast<uintptr_t>(g.next_b) & 15u) == 0) {
    if (!int8_map(&tn, g.next_b, g.next_n, g.next_k, g.next_ld, kN, err)) return -3;
    p.pf_grid = grid_of(g.M, g.next_n, g.next_k);
    p.pf_units = kPrefetchUnits / p.pf_grid;
    p.pf_kblocks = static_cast<int>((g.next_k + kK - 1) / kK);
    p.pf_total = static_cast<int>(next);
  } else {
    tn = tb;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = 1024 + p.stages * (kUnit + a_bytes) + sizeof(Ctl) + kInt8StreamRows * sizeof(float);
  cfg.stream = stream;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = a;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, k_int8_stream, tb, ta, tn, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    *err = std::string("int8 stream launch: ") + cudaGetErrorString(e);
    return -3;
  }
  count_launch();
  return 0;
}

}  // namespace tfb200
