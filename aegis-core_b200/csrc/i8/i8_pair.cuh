#pragma once
// The 8-bit product on CTA pairs (tcgen05 cta_group::2, kind::i8): one
// 256-token x 256-channel tile per pair of SMs, for prompts.
//
// Structure, schedule and teardown are those of umma2_gemm_kernel
// (umma2_kernel.cuh): CTA r loads token rows [m0 + 128r, +128) and channel
// rows [n0 + 128r, +128), 128 codes of K a stage, by plain TMA; the leader
// issues M = 256, N = 256, K = 32 MMAs on both CTAs' tiles; two TMEM
// accumulators let a tile's epilogue overlap the next one's main loop. A stage
// has the bytes of the 16-bit kernel's (32 KB a CTA), and its MMAs take half
// the time, so the copies have half the time to arrive.
//
// The epilogue matters more here: a prompt of a few hundred tokens is one tile a
// pair, whose epilogue nothing hides. Eight warps share it, two for each 32 TMEM
// lanes (tokens), half of the channels each; the tile's channel scales wait in
// shared memory, the next 32 columns are on their way from TMEM while the present
// ones are scaled and stored, 32 bytes a lane and store. With four warps, scales
// from global memory and 16-byte stores it took 6.9 us of a 22.5 us launch
// (256 x 14336 x 4096, B200; 17.4 now).
//
// The leader's last waits, for its peer's arrivals, cost 1 us at the end where tiles come
// from the schedule: a slot is given back behind the peer's stores.
//
// Bound: the tensor cores, and power. B200: 8192^3 357 us (3.1 POP/s, 91% of twice
// the measured bf16 burst rate), 361 to 408 in a long run under the power cap; 2048 x 4096
// x 4096 28.6 us (2.4), two waves of which the second is partly empty; 512 x 4096 x
// 14336 38.5 us, 64 of 148 SMs.
#include "../umma2_kernel.cuh"
#include "i8_common.cuh"
#include "i8_phases.h"

namespace aegis::i8 {

struct PairArgs {
  umma::Args u;  // sizes, raster, schedule, status
  const float* a_scale;
  const float* w_scale;
  const void* bias;
  Out out;
};

inline constexpr int kPairBN = 256, kPairStages = 7;
inline constexpr int kPairEpilogueWarps = 8, kPairThreads = 64 + 32 * kPairEpilogueWarps;
// umma's layout (ring, barriers, schedule), then the tile's channel scales.
struct PairLayout : umma::LayoutPair<kPairBN, kPairStages> {
  using Base = umma::LayoutPair<kPairBN, kPairStages>;
  static constexpr int SCALE_OFF = (Base::BYTES + 15) / 16 * 16;
  static constexpr int ALLOC = SCALE_OFF + kPairBN * 4 + 1024;
  static_assert(ALLOC <= 232448, "a CTA's shared memory");
};

// Arrive on another CTA's mbarrier without waiting for this thread's stores to
// C to be visible in the cluster (a release does: 1 us after a tile's stores). What
// the barrier hands over is TMEM, ordered by the tcgen05 fences.
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Whether `v` holds for every one of `count` threads (whole warps) on hardware barrier `id`.
__device__ __forceinline__ bool named_all(uint32_t id, uint32_t count, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(uint32_t(v)), "r"(id), "r"(count)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// 32 channels of one token: scaled by sa and the scales at `scales` (shared memory),
// plus the bias (one value a lane, for its channel).
__device__ __forceinline__ void scale_chunk(const PairArgs& a, const TokenScale& sa, uint32_t scales, float bias,
                                            const uint32_t (&r)[32], float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const uint4 w = ptx::ld_shared_v4(scales + 4 * i);
    v[i] = scaled(int(r[i]), sa.s, __uint_as_float(w.x));
    v[i + 1] = scaled(int(r[i + 1]), sa.s, __uint_as_float(w.y));
    v[i + 2] = scaled(int(r[i + 2]), sa.s, __uint_as_float(w.z));
    v[i + 3] = scaled(int(r[i + 3]), sa.s, __uint_as_float(w.w));
  }
  if (sa.f != 1.f) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __fmul_rn(v[i], sa.f);
  }
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __fadd_rn(v[i], __shfl_sync(0xffffffffu, bias, i));
  }
}

template <class T>
__device__ __forceinline__ T to_out(float v) {
  if constexpr (sizeof(T) == 2) return Elem<T>::from_f32(v);
  else return v;
}

// A lane's row of C, 32 columns after 32. Where the row does not start on a
// 16-byte boundary (every other row of an odd N, say) the values are shifted to
// the boundaries in registers, the last 16 bytes of a chunk waiting for the next
// one: single 2-byte stores, 32 rows of them an instruction, took four times the
// whole product's time (1000 x 14331 x 4096: 190 us; now 60, the aligned N 50).
template <class T>
struct RowWriter {
  static constexpr int kWords = 32 * int(sizeof(T)) / 4;  // a chunk's
  static constexpr int kVec = 16 / int(sizeof(T));        // values in 16 bytes
  T* at;              // the next column
  int past;           // values since the last 16-byte boundary
  uint32_t carry[4];  // the 16 bytes of values before `at`
  bool begun = false;

  __device__ explicit RowWriter(T* p) : at(p), past(int((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T))) {}

  static __device__ __forceinline__ T value(const uint32_t* w, int i) {
    if constexpr (sizeof(T) == 2) {
      const uint16_t h = uint16_t(w[i >> 1] >> (16 * (i & 1)));
      return reinterpret_cast<const T&>(h);
    } else {
      return reinterpret_cast<const T&>(w[i]);
    }
  }

  __device__ __forceinline__ void chunk(const float (&v)[32]) {
    uint32_t w[4 + kWords + 2];
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      if constexpr (sizeof(T) == 2) w[4 + j] = Elem<T>::pack(v[2 * j], v[2 * j + 1]);
      else w[4 + j] = __float_as_uint(v[j]);
    }
    if ((reinterpret_cast<uintptr_t>(at) & 31u) == 0) {
#pragma unroll
      for (int j = 0; j < kWords; j += 8) {
        const uint32_t o[8] = {w[4 + j], w[5 + j], w[6 + j], w[7 + j], w[8 + j], w[9 + j], w[10 + j], w[11 + j]};
        store32(at + j * (4 / int(sizeof(T))), o);
      }
    } else if (past == 0) {
#pragma unroll
      for (int j = 0; j < kWords; j += 4)
        *reinterpret_cast<uint4*>(at + j * (4 / int(sizeof(T)))) = make_uint4(w[4 + j], w[5 + j], w[6 + j], w[7 + j]);
    } else {
      if (!begun) {  // up to the first boundary
#pragma unroll
        for (int i = 0; i < kVec - 1; ++i)
          if (i < kVec - past) at[i] = value(w + 4, i);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = begun ? carry[j] : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) carry[j] = w[kWords + j];
      w[4 + kWords] = w[5 + kWords] = 0;
      // Values kVec - past on, of those 16 bytes and the chunk.
      int d = kVec - past;
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 4 + kWords; ++j) w[j] = d & 1 ? __funnelshift_r(w[j], w[j + 1], 16) : w[j];
        d >>= 1;
      }
#pragma unroll
      for (int j = 0; j < 4 + kWords; ++j) w[j] = d & 1 ? w[j + 1] : w[j];
#pragma unroll
      for (int j = 0; j < 3 + kWords; ++j) w[j] = d & 2 ? w[j + 2] : w[j];
#pragma unroll
      for (int j = 0; j < kWords; j += 4)
        if (j > 0 || begun)
          *reinterpret_cast<uint4*>(at + j * (4 / int(sizeof(T))) - past) = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
      begun = true;
    }
    at += 32;
  }
  // The values that wait for a chunk that does not come.
  __device__ __forceinline__ void finish() {
    if (begun) {
#pragma unroll
      for (int i = 1; i < kVec; ++i)
        if (i >= kVec - past) at[i - kVec] = value(carry, i);
    }
    begun = false;
  }
};

template <class T>
__global__ void __launch_bounds__(kPairThreads, 1)
    i8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ PairArgs p) {
  using L = PairLayout;
  using umma::Unit;
  constexpr int STAGES = kPairStages;
  const umma::Args& a = p.u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = ptx::smem_addr(smem);
  const int warp = int(threadIdx.x >> 5);
  const int lane = int(threadIdx.x & 31);
  const uint32_t rank = ptx::cluster_ctarank();
  const long long first_unit = blockIdx.x >> 1;

  const uint32_t bar0 = sbase + L::BAR_OFF;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tfull_bar = [&](int acc) { return bar0 + 8u * (2 * STAGES + acc); };
  auto tempty_bar = [&](int acc) { return bar0 + 8u * (2 * STAGES + 2 + acc); };
  const uint32_t drain_bar = bar0 + 8u * (2 * STAGES + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
  const umma::Sched sched{sbase + L::SCHED_OFF, abort_flag, a.status, a.wait_limit_ns};

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full_bar(s), 1);   // the leader's producer; both CTAs' bytes complete it
      ptx::mbar_init(empty_bar(s), 1);  // the leader's commit
    }
    for (int acc = 0; acc < 2; ++acc) {
      ptx::mbar_init(tfull_bar(acc), 1);
      ptx::mbar_init(tempty_bar(acc), 2 * kPairEpilogueWarps);  // one lane a warp, both CTAs
    }
    ptx::mbar_init(drain_bar, 1);
    sched.init(2 * (1 + kPairEpilogueWarps));  // readers: MMA lane and epilogue warps; peer's producer and its
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tensormap(&tmA);
    ptx::prefetch_tensormap(&tmW);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(ptx::smem_addr(tmem_slot), L::TMEM_COLS);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  ptx::cluster_sync();  // both CTAs' barriers exist before any remote arrive or copy
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------ TMA producer (both CTAs)
    int stage = 0;
    uint32_t phase = 0, filled = 0, fill_parity = 0;
    bool ok = true;
    if (lane == 0) {
      umma::SchedOwner owner;
      int seq = 0;
      for (long long unit = first_unit; ok && unit >= 0;) {
        if (rank == 0 && a.steal) owner.request(sched);
        const Unit u = umma::decode_unit_pair<kPairBN>(a, unit);
        const int my_m = u.m0 + 128 * int(rank), my_n = u.n0 + 128 * int(rank);
        for (int i = 0; i < u.nkb; ++i) {
          ok = ptx::mbar_wait_bounded(empty_bar(stage), phase ^ 1u, abort_flag, a.status, kStatusTimeoutProducer,
                                      a.wait_limit_ns);
          if (!ok) break;
          const int k0 = umma::unit_kb(u, i) * BK;
          if (rank == 0) ptx::mbar_arrive_expect_tx(full_bar(stage), 2 * L::STAGE_TX);
          const uint32_t fb = ptx::map_to_rank(full_bar(stage), 0);
          ptx::tma_load_3d_pair(sbase + L::A_OFF + stage * L::A_BYTES, &tmA, fb, k0, my_m, 0);
          ptx::tma_load_3d_pair(sbase + L::B_OFF + stage * L::B_BYTES, &tmW, fb, k0, my_n, 0);
          filled |= 1u << stage;
          fill_parity = (fill_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok || !a.steal) break;  // one tile a pair: no schedule
        ok = rank == 0 ? owner.publish_next(sched, 2, true, &unit, kStatusTimeoutProducer)
                       : umma::sched_take(sched, seq, true, &unit, kStatusTimeoutProducer);
      }
      owner.drain(sched);
      // The leader: every reader has given its slots back, the peer's arrivals for them have landed.
      if (rank == 0 && a.steal && ok)
        for (int i = 0; i < umma::kSchedDepth; ++i)
          if (!ptx::mbar_wait_teardown(sched.empty_bar(i), slot_read(owner.seq, i, umma::kSchedDepth), a.wait_limit_ns) &&
              a.status)
            atomicOr(a.status, kStatusTimeoutDrain);
      for (int s = 0; s < STAGES; ++s)
        if (filled & (1u << s)) {
          const uint32_t par = (fill_parity >> s) & 1u;
          const bool done = rank == 0 ? ptx::mbar_wait_teardown(full_bar(s), par, a.wait_limit_ns)
                                      : ptx::mbar_wait_teardown(empty_bar(s), par, a.wait_limit_ns);
          if (!done && a.status) atomicOr(a.status, kStatusTimeoutDrain);
        }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (leader only)
    if (rank == 0) {
      constexpr uint32_t idesc = idesc_i8(umma::BM_PAIR, kPairBN);
      int stage = 0;
      uint32_t phase = 0;
      AccumulatorTurn turn;
      bool ok = true;
      if (lane == 0) {
        int seq = 0;
        for (long long unit = first_unit; ok && unit >= 0;) {
          const Unit u = umma::decode_unit_pair<kPairBN>(a, unit);
          ok = ptx::mbar_wait_bounded(tempty_bar(turn.acc), turn.read(turn.acc), abort_flag, a.status, kStatusTimeoutMma,
                                      a.wait_limit_ns);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t d_tmem = tmem_base + uint32_t(turn.acc * kPairBN);
          for (int i = 0; i < u.nkb; ++i) {
            ok = ptx::mbar_wait_bounded(full_bar(stage), phase, abort_flag, a.status, kStatusTimeoutMma,
                                        a.wait_limit_ns);
            if (!ok) break;
            ptx::tc_fence_after();
            const uint32_t sa = sbase + L::A_OFF + stage * L::A_BYTES;
            const uint32_t sw = sbase + L::B_OFF + stage * L::B_BYTES;
#pragma unroll
            for (int ks = 0; ks < BK / 32; ++ks) {
              const uint64_t ad = ptx::sdesc_sw128(sa + ks * 32u, 16u, 1024u);
              const uint64_t wd = ptx::sdesc_sw128(sw + ks * 32u, 16u, 1024u);
              umma_i8_pair(d_tmem, ad, wd, idesc, (i > 0 || ks > 0) ? 1u : 0u);
            }
            ptx::umma_commit_pair(empty_bar(stage), 0x3);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          ptx::umma_commit_pair(tfull_bar(turn.acc), 0x3);
          turn.next();
          if (!a.steal) break;
          ok = umma::sched_take(sched, seq, false, &unit, kStatusTimeoutMma);
        }
        // Both accumulators have been read for the last time: the peer's arrivals that say so have landed.
        if (ok)
          for (int acc = 0; acc < 2; ++acc)
            if (!ptx::mbar_wait_teardown(tempty_bar(acc), turn.read(acc), a.wait_limit_ns) && a.status)
              atomicOr(a.status, kStatusTimeoutDrain);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------ epilogue (warps 2..9, both CTAs)
    constexpr int kHalf = kPairBN / 2;
    const int quarter = warp & 3, first = ((warp - 2) >> 2) * kHalf;  // TMEM lanes, first column
    const int et = int(threadIdx.x) - 64;                            // 0..255: the column whose scale it fetches
    const int row_in_tile = 128 * int(rank) + quarter * 32 + lane;
    const uint32_t scales = sbase + L::SCALE_OFF;
    AccumulatorTurn turn;
    bool ok = true;
    int seq = 0;
    for (long long unit = first_unit; ok && unit >= 0;) {
      const Unit u = umma::decode_unit_pair<kPairBN>(a, unit);
      const int row = u.m0 + row_in_tile;
      const bool live = row < a.M;
      const TokenScale sa = token_scale(live ? p.a_scale[row] : 0.f);
      const float sw = u.n0 + et < a.N ? p.w_scale[u.n0 + et] : 0.f;
      float bias[kHalf / 32];
#pragma unroll
      for (int c = 0; c < kHalf / 32; ++c) {
        const int col = u.n0 + first + 32 * c + lane;
        bias[c] = p.bias && col < a.N ? load_as_f32(p.bias, col, p.out) : 0.f;
      }
      ptx::named_barrier(1, 32 * kPairEpilogueWarps);  // the last tile's scales are read
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(scales + 4u * uint32_t(et)), "f"(sw) : "memory");
      ptx::named_barrier(1, 32 * kPairEpilogueWarps);
      if (lane == 0)
        ok = ptx::mbar_wait_bounded(tfull_bar(turn.acc), turn.full(), abort_flag, a.status, kStatusTimeoutEpilogue,
                                    a.wait_limit_ns);
      // One answer for all eight warps: a warp that left alone would strand the others at the barriers.
      ok = named_all(2, 32 * kPairEpilogueWarps, __shfl_sync(0xffffffffu, ok, 0));
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t t_row = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(turn.acc * kPairBN + first);
      RowWriter<T> out(static_cast<T*>(a.C) + (live ? row : 0) * a.ldc + u.n0 + first);
      uint32_t r[2][32];
      ptx::tmem_ld_32x32b_x32(t_row, r[0]);
#pragma unroll
      for (int c = 0; c < kHalf / 32; ++c) {
        ptx::tmem_ld_wait(r[c & 1]);
        if (c + 1 < kHalf / 32) {
          ptx::tmem_ld_32x32b_x32(t_row + 32 * (c + 1), r[(c + 1) & 1]);
        } else {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_relaxed(ptx::map_to_rank(tempty_bar(turn.acc), 0));  // the accumulator is read
        }
        const int col = u.n0 + first + 32 * c;
        if (col >= a.N) continue;
        float v[32];
        scale_chunk(p, sa, scales + 4u * uint32_t(first + 32 * c), bias[c], r[c & 1], v);
        if (!live) continue;
        if (col + 32 <= a.N) {
          out.chunk(v);
        } else {
          out.finish();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (col + i < a.N) out.at[i] = to_out<T>(v[i]);
        }
      }
      if (live) out.finish();
      turn.next();
      if (!a.steal) break;
      long long next = -1;
      if (lane == 0) ok = umma::sched_take(sched, seq, rank != 0, &next, kStatusTimeoutEpilogue);
      ok = named_all(2, 32 * kPairEpilogueWarps, __shfl_sync(0xffffffffu, ok, 0));
      unit = __shfl_sync(0xffffffffu, next, 0);
    }
  }

  // ------------------------------------------------ teardown
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1 && lane == 0) {
    if (rank == 0) ptx::umma_commit_pair(drain_bar, 0x3);
    if (!ptx::mbar_wait_teardown(drain_bar, 0, a.wait_limit_ns) && a.status) atomicOr(a.status, kStatusTimeoutDrain);
  }
  __syncwarp();
  ptx::tc_fence_before();
  // Neither CTA leaves while its peer may still touch its memory. What is sent to the
  // peer's CTA has been waited for there: the leader's slots and accumulators above, the
  // peer's copies on the leader's full barriers, the leader's commits and slots by the
  // peer's roles. After a wait that ran out that is not known, so the barrier itself orders it.
  if (*abort_flag) ptx::cluster_sync();
  else cluster_step();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc_pair(tmem_base, L::TMEM_COLS);
}

}  // namespace aegis::i8
