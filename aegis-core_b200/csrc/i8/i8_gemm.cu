// Host side of the 8-bit product: which kernel, which tiles, the launches.
#include <algorithm>

#include "../gpu_target.h"
#include "../status.h"
#include "../tma_map.h"
#include "i8_align.cuh"
#include "i8_dot.cuh"
#include "i8_pair.cuh"
#include "i8_stream.cuh"

namespace aegis::i8 {

bool tma_rows(const void* p, long long ld, int rows) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (rows <= 1 || ld % 16 == 0);
}

namespace {

// The stream kernel's variants, by tokens a tile. Rings of about 100 KB for up to
// 128 tokens, so two CTAs share an SM and one's epilogue overlaps the other's
// stream; 192 KB for 256. Measured on a B200 (K = 4096, one wave of CTAs): the time
// of a stage, which is the copies' latency over the ring's depth as long as DRAM
// keeps up, and what joining the slices of a cluster costs.
struct StreamVariant {
  int tokens, group, stages, ctas_per_sm;  // group: k-blocks a stage
  double stage_us, join_us;
};
constexpr StreamVariant kStream[] = {
    {16, 2, 3, 2, 0.39, 1.0}, {32, 2, 2, 2, 0.6, 1.3},  {64, 2, 2, 2, 0.77, 1.8},
    {128, 1, 3, 2, 0.58, 2.5}, {256, 1, 4, 1, 0.86, 4.0},
};
constexpr const StreamVariant& variant(int tokens) {
  for (const StreamVariant& v : kStream)
    if (v.tokens == tokens) return v;
  return kStream[0];
}
constexpr int group_for(int nt) { return variant(nt).group; }
constexpr int stages_for(int nt) { return variant(nt).stages; }

}  // namespace

// The estimates below (microseconds) only have to order the choices. Times without what
// every launch costs (about 5). B200, 98 shapes (M = 16 .. 1500; seven layers from 896 x
// 4864 to 4096 x 14336), every tile and cut timed beside the choice: it is within 8% of
// the fastest on 93, 10 to 13% off on four, and 17% on 48 x 1000 x 896 (5.2 us, 4.4).
GemmPlan plan_gemm(int M, int N, int K, int sms) {
  GemmPlan p;
  const int kb = ceil_div(K, BK);
  if (K > 0 && M <= kDotTokens) {
    // Where the loads of a warp's share of K are all on their way at once and no
    // second wave of warps (16 an SM) follows. B200, us, this kernel and the
    // stream kernel: 1 x 4096 x 4096 6.1, 7.5; 4 x 4096 x 4096 6.7, 7.6; 8 x 4096 x
    // 4096 8.4, 7.7; 1 x 896 x 4864 4.1, 5.9; 1 x 4096 x 14336 14.1, 13.0;
    // 1 x 14336 x 4096 17.0, 13.8.
    const long long groups = ceil_div(N, kDotChannels), warps = 16ll * sms;
    int parts = 1;
    while (parts < kDotWarps && groups * parts * 2 <= warps && K >= 1024 * parts) parts *= 2;
    if (groups * parts <= warps && K <= parts * (M <= 4 ? 2048 : 1024)) {
      p.kernel = GemmKernel::Dot;
      p.tile_m = M;
      p.tile_n = kDotChannels;
      p.tiles = groups;
      p.splits = parts;
      p.grid = ceil_div(groups, (long long)(kDotWarps / parts));
      return p;
    }
  }
  // CTA pairs: 256 x 256 tiles, 0.31 us a k-block, and 2.5 more for the first
  // copies and the last epilogue.
  const long long pair_tiles = (long long)ceil_div(M, 256) * ceil_div(N, 256);
  const double dram_us = double(N) * K / 6.5e6;
  double best = 1e300;
  if (K > 0 && M > 64) {
    best = std::max(dram_us, 2.5 + 0.31 * kb * double(ceil_div(pair_tiles, (long long)std::max(1, sms / 2))));
    p.kernel = GemmKernel::Pair;
    p.tile_m = p.tile_n = 256;
    p.tiles = pair_tiles;
    p.grid = 2 * pair_tiles;
  }
  for (const StreamVariant& v : kStream) {
    if (v.tokens > 16 && v.tokens / 2 >= M) break;  // a smaller tile holds them all
    const long long token_tiles = ceil_div(M, v.tokens), slots = (long long)sms * v.ctas_per_sm;
    const int steps = ceil_div(kb, v.group);
    for (int S = 1; S <= 8 && S <= std::max(1, steps); S *= 2) {
      // Clusters of 4 and 8 leave some of a GPC's SMs unused: about an eighth.
      const long long room = S >= 4 ? slots * 7 / 8 : slots;
      int rows = BN;
      long long tiles = token_tiles * ceil_div(N, rows);
      if (S > 1 && tiles * S > room) continue;
      if (S == 1 && tiles < room && dram_us > steps * v.stage_us) {
        // DRAM bounds it: narrower tiles while one wave holds them, so every SM gets the same share.
        const long long each = ceil_div((long long)N, room / token_tiles);
        rows = int(std::min<long long>(BN, (each + 7) / 8 * 8));
        tiles = token_tiles * ceil_div(N, rows);
      }
      const double waves = double(ceil_div(tiles * S, room));
      // Memory: DRAM once, or L2 once a token tile. It hides the stages' time, or the
      // other way round, for the most part. A token's store takes 0.02 us, another wave 3.
      const double memory_us = std::max(dram_us, dram_us * 0.6 * double(token_tiles));
      const double stages_us = waves * ceil_div(steps, S) * v.stage_us;
      const double us = std::max(memory_us, stages_us) + 0.25 * std::min(memory_us, stages_us) +
                        (S > 1 ? v.join_us * (0.9 + 0.1 * double(token_tiles)) : 0.0) + 0.02 * v.tokens + 3.0 * (waves - 1.0);
      if (us < best) {
        best = us;
        p.kernel = GemmKernel::Stream;
        p.tile_m = v.tokens;
        p.tile_n = rows;
        p.splits = S;
        p.tiles = tiles;
        p.grid = tiles * S;
      }
    }
  }
  return p;
}

namespace {

template <int NT>
cudaError_t launch_stream(const CUtensorMap& tw, const CUtensorMap& ta, const StreamArgs& a, unsigned grid,
                          cudaStream_t s) {
  constexpr int ST = stages_for(NT), G = group_for(NT);
  auto* kern = &i8_stream_kernel<NT, ST, G>;
  static gpu::SmemOptIn optin;
  constexpr size_t smem = size_t(StreamLayout<NT, ST, G>::ALLOC);
  if (const cudaError_t e = optin.ensure(reinterpret_cast<const void*>(kern), smem); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kStreamThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits (griddepcontrol.wait)
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(a.splits);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, tw, ta, a);
}

template <int MT>
cudaError_t launch_dot(const DotArgs& a, unsigned grid, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kDotThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits (griddepcontrol.wait)
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, &i8_dot_kernel<MT>, a);
}
cudaError_t launch_dot(const DotArgs& a, unsigned grid, cudaStream_t s) {
  if (a.M == 1) return launch_dot<1>(a, grid, s);
  if (a.M == 2) return launch_dot<2>(a, grid, s);
  if (a.M <= 4) return launch_dot<4>(a, grid, s);
  return launch_dot<8>(a, grid, s);
}

cudaError_t launch_stream(int nt, const CUtensorMap& tw, const CUtensorMap& ta, const StreamArgs& a, unsigned grid,
                          cudaStream_t s) {
  switch (nt) {
    case 16: return launch_stream<16>(tw, ta, a, grid, s);
    case 32: return launch_stream<32>(tw, ta, a, grid, s);
    case 64: return launch_stream<64>(tw, ta, a, grid, s);
    case 128: return launch_stream<128>(tw, ta, a, grid, s);
    default: return launch_stream<256>(tw, ta, a, grid, s);
  }
}

template <class T>
cudaError_t launch_pair(const CUtensorMap& ta, const CUtensorMap& tw, const PairArgs& a, unsigned grid,
                        cudaStream_t s) {
  auto* kern = &i8_pair_kernel<T>;
  static gpu::SmemOptIn optin;
  constexpr size_t smem = size_t(PairLayout::ALLOC);
  if (const cudaError_t e = optin.ensure(reinterpret_cast<const void*>(kern), smem); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, ta, tw, a);
}

constexpr long long kMaxPairUnits = 1ll << 29;  // umma's raster arithmetic is 32-bit

// Rows that TMA can address as they are, or a copy of them.
struct Rows {
  const void* p;
  long long ld;
  int K;
};
// Copies of W (N rows) and of A (M rows), where asked for, in one launch.
cudaError_t align_rows(Rows* w, int N, void* w_copy, Rows* t, int M, void* t_copy, cudaStream_t s) {
  AlignArgs a{};
  a.K = w_copy ? w->K : t->K;
  a.padded = int(aligned_cols(a.K));
  a.segments = ceil_div(a.padded, 128 * kAlignWords);
  if (w_copy) a.job[0] = {static_cast<const int8_t*>(w->p), w->ld, static_cast<int8_t*>(w_copy), (long long)N * a.segments};
  if (t_copy) a.job[1] = {static_cast<const int8_t*>(t->p), t->ld, static_cast<int8_t*>(t_copy), (long long)M * a.segments};
  const long long grid = ceil_div(a.job[0].tasks + a.job[1].tasks, (long long)(kAlignThreads / 32));
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  if (w_copy) *w = Rows{w_copy, a.padded, a.padded};
  if (t_copy) *t = Rows{t_copy, a.padded, a.padded};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kAlignThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits (griddepcontrol.wait)
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, &i8_align_kernel, a);
}

}  // namespace

cudaError_t align(const void* src, long long ld, int rows, int K, void* dst, cudaStream_t s) {
  Rows r{src, ld, K};
  return align_rows(&r, rows, dst, nullptr, 0, nullptr, s);
}

GemmSpace gemm_space(const void* A, long long lda, const void* W, long long ldw, int M, int N, int K) {
  GemmSpace sp;
  sp.w = K > 0 && !tma_rows(W, ldw, N) ? size_t(N) * aligned_cols(K) : 0;
  sp.a = K > 0 && !tma_rows(A, lda, M) ? size_t(M) * aligned_cols(K) : 0;
  return sp;
}

cudaError_t gemm(const Gemm& g, cudaStream_t s) {
  if (g.M == 0 || g.N == 0) return cudaSuccess;
  const gpu::Target* d = gpu::this_device();
  if (!d || d->cc != 100) return cudaErrorNotSupported;
  unsigned* status = nullptr;
  if (const cudaError_t e = status::word(&status); e != cudaSuccess) return e;
  const GemmPlan p = plan_gemm(g.M, g.N, g.K, d->sms);
  // Copies of rows that TMA cannot address: the weights' first, then the tokens'.
  // A single row's stride means nothing: a tensor map gets one that it can hold.
  const long long one = (long long)aligned_cols(std::max(g.K, 1));
  Rows ra{g.A, g.M > 1 ? g.lda : one, g.K}, rw{g.W, g.N > 1 ? g.ldw : one, g.K};
  const GemmSpace space = gemm_space(g.A, g.lda, g.W, g.ldw, g.M, g.N, g.K);
  char* ws = static_cast<char*>(g.workspace);
  if (space.w || space.a)
    if (const cudaError_t e = align_rows(&rw, g.N, space.w ? ws : nullptr, &ra, g.M, space.a ? ws + space.w : nullptr, s);
        e != cudaSuccess)
      return e;
  const bool settled = g.weights_settled && !space.w;  // a copy of the weights is not there before its kernel has ended
  CUtensorMap ta{}, tw{};
  const int group = p.kernel == GemmKernel::Stream ? group_for(p.tile_m) : 1;
  // Rows of whole k-blocks: a box may take several (one copy a stage; elsewhere
  // the tail of a shorter last one would reach past the rows' end).
  const bool cubes_a = group > 1 && ra.K % BK == 0, cubes_w = group > 1 && rw.K % BK == 0;
  if (g.K > 0 && p.kernel != GemmKernel::Dot &&
      (!encode_map_i8(&ta, ra.p, ra.K, g.M, ra.ld, p.kernel == GemmKernel::Pair ? 128 : p.tile_m, cubes_a ? group : 0) ||
       !encode_map_i8(&tw, rw.p, rw.K, g.N, rw.ld, p.kernel == GemmKernel::Pair ? 128 : p.tile_n, cubes_w ? group : 0)))
    return cudaErrorInvalidValue;  // the driver refused the geometry
  if (p.kernel == GemmKernel::Pair) {
    if (p.tiles > kMaxPairUnits) return cudaErrorInvalidValue;
    PairArgs a{};
    a.u.M = g.M;
    a.u.N = g.N;
    a.u.K = g.K;
    a.u.batch = 1;
    a.u.tiles_m = ceil_div(g.M, 256);
    a.u.tiles_n = ceil_div(g.N, 256);
    a.u.group_m = 8;
    a.u.steal = p.tiles > d->sms / 2;
    a.u.splits = 1;
    a.u.kb_total = a.u.kb_per_split = ceil_div(g.K, BK);
    a.u.units = p.tiles;
    a.u.C = g.C;
    a.u.ldc = g.ldc;
    a.u.status = status;
    a.u.wait_limit_ns = kDefaultWaitLimitNs;
    a.a_scale = g.a_scale;
    a.w_scale = g.w_scale;
    a.bias = g.bias;
    a.out = g.out;
    const unsigned grid = unsigned(p.grid);
    if (g.out == Out::F32) return launch_pair<float>(ta, tw, a, grid, s);
    if (g.out == Out::BF16) return launch_pair<__nv_bfloat16>(ta, tw, a, grid, s);
    return launch_pair<__half>(ta, tw, a, grid, s);
  }
  if (p.grid > 0x7fffffffll) return cudaErrorInvalidValue;
  if (p.kernel == GemmKernel::Dot) {
    DotArgs a{};
    a.M = g.M;
    a.N = g.N;
    a.K = g.K;
    a.parts = p.splits;
    a.weights_early = settled;
    a.A = static_cast<const int8_t*>(ra.p);
    a.W = static_cast<const int8_t*>(rw.p);
    a.lda = ra.ld;
    a.ldw = rw.ld;
    a.ldc = g.ldc;
    a.a_scale = g.a_scale;
    a.w_scale = g.w_scale;
    a.bias = g.bias;
    a.C = g.C;
    a.out = g.out;
    return launch_dot(a, unsigned(p.grid), s);
  }
  StreamArgs a{};
  a.M = g.M;
  a.N = g.N;
  a.K = g.K;
  a.steps = ceil_div(g.K, BK * group);
  a.cubes_w = cubes_w;
  a.cubes_a = cubes_a;
  a.token_tiles = ceil_div(g.M, p.tile_m);
  a.splits = p.splits;
  a.weights_early = settled;
  a.rows = p.tile_n;
  a.ldc = g.ldc;
  a.a_scale = g.a_scale;
  a.w_scale = g.w_scale;
  a.bias = g.bias;
  a.C = g.C;
  a.out = g.out;
  a.status = status;
  a.wait_limit_ns = kDefaultWaitLimitNs;
  return launch_stream(p.tile_m, tw, ta, a, unsigned(p.grid), s);
}

}  // namespace aegis::i8
