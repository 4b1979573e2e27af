#pragma once
// The stream kernel of the 8-bit product: C^T[n, m] = W[n, :] . A[m, :], the
// weights as the 128-row tcgen05 operand and NT tokens as the other (kind::i8,
// M = 128, N = NT, K = 32, int32 accumulators in TMEM), so a decode step's few
// tokens cost no tensor rows and the kernel is a stream of weights.
//
// One CTA computes one slice of K of one 128-channel x NT-token tile:
//   warp 0      TMA producer: a STAGES-deep ring of G k-blocks each (weights
//               16 KB, tokens NT * 128 B a k-block);
//   warp 1      allocates TMEM, issues the MMAs (one lane);
//   warps 2..5  epilogue.
// The `splits` CTAs of a tile form one thread-block cluster. Each leaves its
// int32 sums in its own shared memory (the ring, which is free by then), and
// after a cluster barrier every CTA adds up an equal share of the tokens over
// distributed shared memory, scales and stores it. Whole numbers add up the
// same in any order: the result does not depend on the split. No workspace,
// tickets or atomics, so concurrent calls and captured graphs share nothing.
//
// Bound: the weights from DRAM, and about 5 us a launch in which DRAM is not busy
// (the end of the last grid to this one's wait 1.4, first copies 1.2, joining and the
// tail). B200, cold L2, us: 16 x 4096 x 4096 7.4 (2.3 TB/s), 16 x 14336 x 4096 14.2
// (4.2), 16 x 28672 x 4096 21.5 (5.5). Two CTAs an SM fill its shared memory; smaller
// rings, with which the next launch's CTAs fit beside these, were 2 to 14% slower.
//
// Every wait is bounded; on expiry the CTA records a status bit, its roles
// stop waiting, and it still passes the cluster barriers and frees its TMEM.
#include "i8_common.cuh"

namespace aegis::i8 {

struct StreamArgs {
  int M, N, K;
  int steps;         // stages' worth of K (G k-blocks each) of the whole sum
  int cubes_w, cubes_a;  // rows of whole k-blocks: the tensor map's third coordinate counts them
  int rows;          // channels a tile: a multiple of 8, BN at most
  int token_tiles;   // tiles along the tokens (fastest in the grid, so they share weights in L2)
  int splits;        // cluster size
  int weights_early; // read weights before the grid this one depends on has completed
  long long ldc;
  const float* a_scale;
  const float* w_scale;
  const void* bias;
  void* C;
  Out out;
  unsigned* status;
  long long wait_limit_ns;
};

inline constexpr int kStreamThreads = 192;
inline constexpr int BN = 128;  // channels a tile (MMA M), at most

template <int NT, int STAGES, int G>
struct StreamLayout {
  // [k-block][channel][128], `rows` channels; the MMAs read BN rows from each
  // block's start on, the last ones of them whatever lies there, for TMEM lanes that are not stored.
  static constexpr int W_BYTES = BN * BK * G;
  static constexpr int A_BYTES = NT * BK * G;
  static constexpr int A_OFF = STAGES * W_BYTES;
  static constexpr int RING = STAGES * (W_BYTES + A_BYTES);
  static constexpr int BAR_OFF = RING;
  static constexpr int NBARS = 2 * STAGES + 2;  // full[S], empty[S], done, drain
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  static constexpr int BYTES = MISC_OFF + 16;
  static constexpr int ALLOC = BYTES + 1024;
  static constexpr int TMEM_COLS = NT < 32 ? 32 : NT;
  static_assert(A_BYTES % 1024 == 0, "operand tiles stay 1024-byte aligned");
  static_assert(NT * BN * 4 <= RING, "the int32 tile of a split fits the ring");
};

template <int NT, int STAGES, int G>
__global__ void __launch_bounds__(kStreamThreads, 1)
    i8_stream_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                     const __grid_constant__ StreamArgs a) {
  using L = StreamLayout<NT, STAGES, G>;
  constexpr int BKS = BK * G;  // codes of K a stage
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = ptx::smem_addr(smem);
  const int warp = int(threadIdx.x >> 5), lane = int(threadIdx.x & 31);
  const uint32_t bar0 = sbase + L::BAR_OFF;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  const uint32_t done_bar = bar0 + 8u * (2 * STAGES);
  const uint32_t drain_bar = bar0 + 8u * (2 * STAGES + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);

  const unsigned split = blockIdx.x % unsigned(a.splits);
  const unsigned tile = blockIdx.x / unsigned(a.splits);
  const int m0 = int(tile % unsigned(a.token_tiles)) * NT;
  const int n0 = int(tile / unsigned(a.token_tiles)) * a.rows;
  const int n_end = min(a.N, n0 + a.rows);
  const int w_block = a.rows * BK;  // bytes of a k-block of weights
  const uint32_t stage_bytes = uint32_t(w_block * G + L::A_BYTES);
  const int kb0 = int((long long)a.steps * split / a.splits);  // in stages
  const int nkb = int((long long)a.steps * (split + 1) / a.splits) - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(done_bar, 1);
    ptx::mbar_init(drain_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    if (nkb > 0) {
      ptx::prefetch_tensormap(&tmW);
      ptx::prefetch_tensormap(&tmA);
    }
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_addr(tmem_slot), L::TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // One stage's box of `rows` rows: one copy where the map counts k-blocks, else one a k-block.
  auto copy_box = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int step, int row0, int box_bytes, int cubes) {
    if (cubes) {
      ptx::tma_load_3d(dst, map, bar, 0, row0, step * G);
    } else {
#pragma unroll
      for (int j = 0; j < G; ++j) ptx::tma_load_3d(dst + j * box_bytes, map, bar, (step * G + j) * BK, row0, 0);
    }
  };
  int early = 0;  // stages whose weights are already on their way
  if (warp == 0 && lane == 0) {
    if (a.weights_early) {
      for (const int n = min(nkb, STAGES); early < n; ++early) {
        ptx::mbar_arrive_expect_tx(full_bar(early), stage_bytes);
        copy_box(sbase + early * L::W_BYTES, &tmW, full_bar(early), kb0 + early, n0, w_block, a.cubes_w);
      }
    } else if (a.cubes_w) {
      // Hints (ptx::tma_prefetch_3d): the copies proper follow the wait. Deeper
      // ones, up to 64 MB in all, measured level to 20% slower.
      for (int i = 0; i < min(nkb, STAGES); ++i) ptx::tma_prefetch_3d(&tmW, 0, n0, (kb0 + i) * G);
    }
  }
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t filled = 0, fill_parity = 0;
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < nkb; ++i) {
        const uint32_t fb = full_bar(stage);
        if (i >= early) {
          if (!ptx::mbar_wait_bounded(empty_bar(stage), phase ^ 1u, abort_flag, a.status, kStatusTimeoutProducer,
                                      a.wait_limit_ns))
            break;
          ptx::mbar_arrive_expect_tx(fb, stage_bytes);
          copy_box(sbase + stage * L::W_BYTES, &tmW, fb, kb0 + i, n0, w_block, a.cubes_w);
        }
        copy_box(sbase + L::A_OFF + stage * L::A_BYTES, &tmA, fb, kb0 + i, m0, NT * BK, a.cubes_a);
        filled |= 1u << stage;
        fill_parity = (fill_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // Every copy has landed before the ring is used for anything else.
      for (int s = 0; s < STAGES; ++s)
        if (filled & (1u << s))
          if (!ptx::mbar_wait_teardown(full_bar(s), (fill_parity >> s) & 1u, a.wait_limit_ns) && a.status)
            atomicOr(a.status, kStatusTimeoutDrain);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8(BN, NT);
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < nkb; ++i) {
        if (!ptx::mbar_wait_bounded(full_bar(stage), phase, abort_flag, a.status, kStatusTimeoutMma, a.wait_limit_ns))
          break;
        ptx::tc_fence_after();
        const uint32_t sw = sbase + stage * L::W_BYTES;
        const uint32_t sa = sbase + L::A_OFF + stage * L::A_BYTES;
#pragma unroll
        for (int ks = 0; ks < BKS / 32; ++ks) {
          const uint64_t wd = ptx::sdesc_sw128(sw + (ks / 4) * w_block + (ks % 4) * 32u, 16u, 1024u);
          const uint64_t ad = ptx::sdesc_sw128(sa + (ks / 4) * (NT * BK) + (ks % 4) * 32u, 16u, 1024u);
          umma_i8(tmem_base, wd, ad, idesc, (i > 0 || ks > 0) ? 1u : 0u);
        }
        ptx::umma_commit(empty_bar(stage));
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      ptx::umma_commit(done_bar);
    }
    __syncwarp();
  }

  // ---------------------------------------------------------------- epilogue
  const int mt = min(NT, a.M - m0);  // tokens of this tile
  if (warp >= 2) {
    const int quarter = warp & 3;
    const int n = n0 + quarter * 32 + lane;
    bool ok = true;
    if (nkb > 0) {
      if (lane == 0)
        ok = ptx::mbar_wait_bounded(done_bar, 0, abort_flag, a.status, kStatusTimeoutEpilogue, a.wait_limit_ns);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      ptx::tc_fence_after();
    }
    const uint32_t t_row = tmem_base + (uint32_t(quarter * 32) << 16);
    const bool live = n < n_end;
    const float sw = live ? a.w_scale[n] : 0.f;
    const float b = live && a.bias ? load_as_f32(a.bias, n, a.out) : 0.f;
    constexpr int CH = NT < 32 ? NT : 32;
    for (int c = 0; c < mt && ok; c += CH) {
      uint32_t r[CH];
      if constexpr (CH == 16) ptx::tmem_ld_32x32b_x16(t_row + c, r);
      else ptx::tmem_ld_32x32b_x32(t_row + c, r);
      ptx::tmem_ld_wait(r);
      if (nkb == 0)
#pragma unroll
        for (int j = 0; j < CH; ++j) r[j] = 0;
      if (a.splits == 1) {
        if (live)
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            if (c + j >= mt) break;
            const TokenScale sa = token_scale(a.a_scale[m0 + c + j]);
            const float v = a.bias ? scaled(int(r[j]), sa, sw, b) : scaled(int(r[j]), sa, sw);
            store_one(a.C, (long long)(m0 + c + j) * a.ldc + n, v, a.out);
          }
      } else {
        int* mine = reinterpret_cast<int*>(smem) + quarter * 32 + lane;
#pragma unroll
        for (int j = 0; j < CH; ++j)
          if (c + j < mt) mine[(c + j) * BN] = int(r[j]);
      }
    }
  }
  // The accumulator is read: TMEM goes back while the slices are joined. Every
  // MMA has finished, unless the CTA gave up waiting.
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    if (*abort_flag) {
      if (lane == 0) {
        ptx::umma_commit(drain_bar);
        if (!ptx::mbar_wait_teardown(drain_bar, 0, a.wait_limit_ns) && a.status)
          atomicOr(a.status, kStatusTimeoutDrain);
      }
      __syncwarp();
    }
    ptx::tmem_dealloc(tmem_base, L::TMEM_COLS);
  }
  if (a.splits > 1) {
    __syncwarp();
    ptx::cluster_sync();  // every slice's sums are in its CTA's shared memory
    // This CTA's share: tokens [t0, t1), 32 pieces of 4 channels each.
    const int t0 = int((long long)mt * split / a.splits), t1 = int((long long)mt * (split + 1) / a.splits);
    const bool gone = *abort_flag != 0;  // recorded; this tile's results are not valid
    for (int i = int(threadIdx.x); i < (t1 - t0) * 32 && !gone; i += kStreamThreads) {
      const int t = t0 + (i >> 5), nl = (i & 31) * 4;
      const uint32_t at = sbase + uint32_t((t * BN + nl) * 4);
      int4 sum = make_int4(0, 0, 0, 0);
      for (int q = 0; q < a.splits; ++q) {
        const int4 v = ld_cluster_v4(ptx::map_to_rank(at, q));
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
      const TokenScale sa = token_scale(a.a_scale[m0 + t]);
      const int acc[4] = {sum.x, sum.y, sum.z, sum.w};
      const int n = n0 + nl;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < n_end) {
          const float sw = a.w_scale[n + j];
          const float v = a.bias ? scaled(acc[j], sa, sw, load_as_f32(a.bias, n + j, a.out)) : scaled(acc[j], sa, sw);
          store_one(a.C, (long long)(m0 + t) * a.ldc + n + j, v, a.out);
        }
    }
  }

  if (a.splits > 1) {
    __syncwarp();
    cluster_step();  // no CTA leaves while a peer may still read its sums
  }
}

}  // namespace aegis::i8
