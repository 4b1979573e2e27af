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
// the time, so the copies have half the time to arrive. Here the epilogue
// scales the int32 sums: a lane has one token (its scale in a register), the
// 32 channels of a chunk share their scales across the lanes.
#include "../umma2_kernel.cuh"
#include "i8_common.cuh"

namespace aegis::i8 {

struct PairArgs {
  umma::Args u;  // sizes, raster, schedule, status
  const float* a_scale;
  const float* w_scale;
  const void* bias;
  Out out;
};

inline constexpr int kPairBN = 256, kPairStages = 7;
using PairLayout = umma::LayoutPair<kPairBN, kPairStages>;

// 32 channels of one token: scaled, rounded, stored (ncols of them).
template <class T>
__device__ __forceinline__ void store_chunk(const PairArgs& a, long long row, int col, float sa, const uint32_t (&r)[32]) {
  const int ncols = min(32, a.u.N - col);
  float v[32];
  if (ncols == 32 && (reinterpret_cast<uintptr_t>(a.w_scale) & 15u) == 0) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 sw = __ldg(reinterpret_cast<const float4*>(a.w_scale + col + i));
      v[i] = scaled(int(r[i]), sa, sw.x);
      v[i + 1] = scaled(int(r[i + 1]), sa, sw.y);
      v[i + 2] = scaled(int(r[i + 2]), sa, sw.z);
      v[i + 3] = scaled(int(r[i + 3]), sa, sw.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = i < ncols ? scaled(int(r[i]), sa, __ldg(a.w_scale + col + i)) : 0.f;
  }
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < ncols) v[i] = __fadd_rn(v[i], load_as_f32(a.bias, col + i, a.out));
  }
  T* dst = static_cast<T*>(a.u.C) + row * a.u.ldc + col;
  if constexpr (sizeof(T) == 2) {
    umma::store_row_chunk<T>(dst, v, ncols);
  } else {
    if (ncols == 32 && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
#pragma unroll
      for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < ncols) dst[i] = v[i];
    }
  }
}

template <class T>
__global__ void __launch_bounds__(umma::kThreads, 1)
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
      ptx::mbar_init(tempty_bar(acc), 256);  // every epilogue thread of both CTAs
    }
    ptx::mbar_init(drain_bar, 1);
    sched.init(10);  // 1 + 4 readers in the leader, 1 + 4 in the peer
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tensormap(&tmA);
    ptx::prefetch_tensormap(&tmW);
    // The weights of the first k-blocks into L2 while the previous grid ends
    // (a hint, see ptx::tma_prefetch_3d); the tokens are often its output.
    const Unit u = umma::decode_unit_pair<kPairBN>(a, first_unit);
    const int wn = u.n0 + 128 * int(rank);
    for (int i = 0; i < min(u.nkb, STAGES); ++i)
      if (wn + 128 <= a.N && (i + 1) * BK <= a.K) ptx::tma_prefetch_3d(&tmW, i * BK, wn, 0);
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
        if (!ok) break;
        ok = rank == 0 ? owner.publish_next(sched, 2, true, &unit, kStatusTimeoutProducer)
                       : umma::sched_take(sched, seq, true, &unit, kStatusTimeoutProducer);
      }
      owner.drain(sched);
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
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      if (lane == 0) {
        int seq = 0;
        for (long long unit = first_unit; ok && unit >= 0;) {
          const Unit u = umma::decode_unit_pair<kPairBN>(a, unit);
          ok = ptx::mbar_wait_bounded(tempty_bar(acc), acc_phase ^ 1u, abort_flag, a.status, kStatusTimeoutMma,
                                      a.wait_limit_ns);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t d_tmem = tmem_base + uint32_t(acc * kPairBN);
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
          ptx::umma_commit_pair(tfull_bar(acc), 0x3);
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1u;
          ok = umma::sched_take(sched, seq, false, &unit, kStatusTimeoutMma);
        }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------------------------ epilogue (warps 2..5, both CTAs)
    const int quarter = warp & 3;
    const int row_in_tile = 128 * int(rank) + quarter * 32 + lane;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    int seq = 0;
    for (long long unit = first_unit; ok && unit >= 0;) {
      const Unit u = umma::decode_unit_pair<kPairBN>(a, unit);
      const int row = u.m0 + row_in_tile;
      const float sa = row < a.M ? __ldg(p.a_scale + row) : 0.f;
      if (lane == 0)
        ok = ptx::mbar_wait_bounded(tfull_bar(acc), acc_phase, abort_flag, a.status, kStatusTimeoutEpilogue,
                                    a.wait_limit_ns);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t t_row = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(acc * kPairBN);
      for (int c = 0; c < kPairBN && u.n0 + c < a.N; c += 32) {
        uint32_t r[32];
        ptx::tmem_ld_32x32b_x32(t_row + c, r);
        ptx::tmem_ld_wait(r);
        if (row < a.M) store_chunk<T>(p, row, u.n0 + c, sa, r);
      }
      ptx::tc_fence_before();
      ptx::mbar_arrive_cluster(ptx::map_to_rank(tempty_bar(acc), 0));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
      long long next = -1;
      if (lane == 0) ok = umma::sched_take(sched, seq, rank != 0, &next, kStatusTimeoutEpilogue);
      ok = __shfl_sync(0xffffffffu, ok, 0);
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
  ptx::cluster_sync();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc_pair(tmem_base, L::TMEM_COLS);
}

}  // namespace aegis::i8
