#pragma once
// The stream kernel of the 8-bit product: C^T[n, m] = W[n, :] . A[m, :], the
// weights as the 128-row tcgen05 operand and NT tokens as the other (kind::i8,
// M = 128, N = NT, K = 32, int32 accumulators in TMEM), so a decode step's few
// tokens cost no tensor rows and the kernel is a stream of weights.
//
// One CTA computes one slice of K of one 128-channel x NT-token tile:
//   warp 0      TMA producer: a STAGES-deep ring of (weights 16 KB, tokens
//               NT * 128 B) k-blocks;
//   warp 1      allocates TMEM, issues the MMAs (one lane);
//   warps 2..5  epilogue; with kLoadThreads they also fill the ring, 16 bytes
//               at a time, for operands whose rows TMA cannot address.
// The `splits` CTAs of a tile form one thread-block cluster. Each leaves its
// int32 sums in its own shared memory (the ring, which is free by then), and
// after a cluster barrier every CTA adds up an equal share of the tokens over
// distributed shared memory, scales and stores it. Whole numbers add up the
// same in any order: the result does not depend on the split. No workspace,
// tickets or atomics, so concurrent calls and captured graphs share nothing.
//
// Every wait is bounded; on expiry the CTA records a status bit, its roles
// stop waiting, and it still passes the cluster barriers and frees its TMEM.
#include "i8_common.cuh"

namespace aegis::i8 {

enum Load : int { kLoadTma = 0, kLoadThreads = 1 };

struct StreamArgs {
  int M, N, K;
  int kb;            // k-blocks of the whole sum
  int token_tiles;   // tiles along the tokens (fastest in the grid, so they share weights in L2)
  int splits;        // cluster size
  int weights_early; // read weights before the grid this one depends on has completed
  const int8_t* A;
  const int8_t* W;
  long long lda, ldw, ldc;
  const float* a_scale;
  const float* w_scale;
  const void* bias;
  void* C;
  Out out;
  unsigned* status;
  long long wait_limit_ns;
};

inline constexpr int kStreamThreads = 192;
inline constexpr int BN = 128;  // channels a tile (MMA M)

template <int NT, int STAGES>
struct StreamLayout {
  static constexpr int W_BYTES = BN * BK;
  static constexpr int A_BYTES = NT * BK;
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

// 16 codes of a row from any byte address; bytes at or beyond `left` are zero.
// Whole pieces are read as aligned 32-bit words (each holds at least one byte
// of the piece) and shifted together; a row's last piece is read by bytes.
__device__ __forceinline__ uint4 load_piece(const int8_t* p, long long left) {
  uint32_t v[4] = {0, 0, 0, 0};
  if (left >= 16) {
    const uint32_t mis = uint32_t(reinterpret_cast<uintptr_t>(p) & 3u);
    const uint32_t* q = reinterpret_cast<const uint32_t*>(p - mis);
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __ldg(q + i);
    w[4] = mis ? __ldg(q + 4) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __funnelshift_r(w[i], w[i + 1], mis * 8u);
  } else {
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (i < left) v[i >> 2] |= uint32_t(uint8_t(__ldg(p + i))) << (8 * (i & 3));
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// `rows` rows x 128 codes of a row-major matrix into a 128-byte-swizzled tile
// at shared address `dst`, by 128 threads; rows from `limit` on and codes from
// column K on are zero.
__device__ __forceinline__ void fill_tile(uint32_t dst, const int8_t* base, long long ld, int row0, int rows, int limit,
                                          int k0, int K, int tid) {
#pragma unroll 4
  for (int i = tid; i < rows * 8; i += 128) {
    const int r = i >> 3, c = i & 7;
    const int row = row0 + r, k = k0 + 16 * c;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < limit && k < K) v = load_piece(base + (long long)row * ld + k, K - k);
    ptx::st_shared_v4(dst + uint32_t(r * 128 + ((c ^ (r & 7)) * 16)), v.x, v.y, v.z, v.w);
  }
}

template <int NT, int STAGES, int LOAD>
__global__ void __launch_bounds__(kStreamThreads, 1)
    i8_stream_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                     const __grid_constant__ StreamArgs a) {
  using L = StreamLayout<NT, STAGES>;
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
  const int n0 = int(tile / unsigned(a.token_tiles)) * BN;
  const int kb0 = int((long long)a.kb * split / a.splits);
  const int nkb = int((long long)a.kb * (split + 1) / a.splits) - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full_bar(s), LOAD == kLoadTma ? 1 : 128);
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(done_bar, 1);
    ptx::mbar_init(drain_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    if (LOAD == kLoadTma) {
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

  int early = 0;  // k-blocks whose weights are already on their way
  if (LOAD == kLoadTma && warp == 0 && lane == 0) {
    const int n = min(nkb, STAGES);
    if (a.weights_early) {
      for (; early < n; ++early) {
        ptx::mbar_arrive_expect_tx(full_bar(early), L::W_BYTES + L::A_BYTES);
        ptx::tma_load_3d(sbase + early * L::W_BYTES, &tmW, full_bar(early), (kb0 + early) * BK, n0, 0);
      }
    } else {
      // A hint only (ptx::tma_prefetch_3d): the copies proper follow the wait.
      for (int i = 0; i < n; ++i)
        if (n0 + BN <= a.N && (kb0 + i + 1) * BK <= a.K) ptx::tma_prefetch_3d(&tmW, (kb0 + i) * BK, n0, 0);
    }
  }
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();

  if (warp == 0) {
    if (LOAD == kLoadTma && lane == 0) {
      uint32_t filled = 0, fill_parity = 0;
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < nkb; ++i) {
        const uint32_t fb = full_bar(stage);
        if (i >= early) {
          if (!ptx::mbar_wait_bounded(empty_bar(stage), phase ^ 1u, abort_flag, a.status, kStatusTimeoutProducer,
                                      a.wait_limit_ns))
            break;
          ptx::mbar_arrive_expect_tx(fb, L::W_BYTES + L::A_BYTES);
          ptx::tma_load_3d(sbase + stage * L::W_BYTES, &tmW, fb, (kb0 + i) * BK, n0, 0);
        }
        ptx::tma_load_3d(sbase + L::A_OFF + stage * L::A_BYTES, &tmA, fb, (kb0 + i) * BK, m0, 0);
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
        for (int ks = 0; ks < BK / 32; ++ks) {
          const uint64_t wd = ptx::sdesc_sw128(sw + ks * 32u, 16u, 1024u);
          const uint64_t ad = ptx::sdesc_sw128(sa + ks * 32u, 16u, 1024u);
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
  } else if (LOAD == kLoadThreads) {
    const int tid = int(threadIdx.x) - 64;
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < nkb; ++i) {
      if (!ptx::mbar_wait_bounded(empty_bar(stage), phase ^ 1u, abort_flag, a.status, kStatusTimeoutProducer,
                                  a.wait_limit_ns))
        break;
      const int k0 = (kb0 + i) * BK;
      fill_tile(sbase + stage * L::W_BYTES, a.W, a.ldw, n0, BN, a.N, k0, a.K, tid);
      fill_tile(sbase + L::A_OFF + stage * L::A_BYTES, a.A, a.lda, m0, NT, a.M, k0, a.K, tid);
      fence_proxy_async();
      ptx::mbar_arrive(full_bar(stage));
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
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
    const bool live = n < a.N;
    const float sw = live ? __ldg(a.w_scale + n) : 0.f;
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
            const float sa = __ldg(a.a_scale + m0 + c + j);
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
      const float sa = __ldg(a.a_scale + m0 + t);
      const int acc[4] = {sum.x, sum.y, sum.z, sum.w};
      const int n = n0 + nl;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < a.N) {
          const float sw = __ldg(a.w_scale + n + j);
          const float v = a.bias ? scaled(acc[j], sa, sw, load_as_f32(a.bias, n + j, a.out)) : scaled(acc[j], sa, sw);
          store_one(a.C, (long long)(m0 + t) * a.ldc + n + j, v, a.out);
        }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    if (lane == 0) {
      ptx::umma_commit(drain_bar);
      if (!ptx::mbar_wait_teardown(drain_bar, 0, a.wait_limit_ns) && a.status) atomicOr(a.status, kStatusTimeoutDrain);
    }
    __syncwarp();
    ptx::tmem_dealloc(tmem_base, L::TMEM_COLS);
  }
  if (a.splits > 1) ptx::cluster_sync();  // no CTA leaves while a peer may still read its sums
}

}  // namespace aegis::i8
