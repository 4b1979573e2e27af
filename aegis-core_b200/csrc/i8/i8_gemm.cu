// Host side of the 8-bit product: which kernel, which tiles, the launches.
#include <algorithm>

#include "../gpu_target.h"
#include "../status.h"
#include "../tma_map.h"
#include "i8_pair.cuh"
#include "i8_stream.cuh"

namespace aegis::i8 {

bool tma_rows(const void* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 16 == 0; }

namespace {

// Ring depths: about 100 KB for up to 128 tokens, so two CTAs share an SM and
// one's epilogue overlaps the other's stream; 192 KB for 256 tokens.
constexpr int stages_for(int nt) { return nt == 16 ? 6 : nt == 32 ? 5 : nt == 64 ? 4 : nt == 128 ? 3 : 4; }
constexpr int ctas_per_sm(int nt) { return nt <= 128 ? 2 : 1; }

}  // namespace

GemmPlan plan_gemm(int M, int N, int K, bool tma, int sms) {
  GemmPlan p;
  const int kb = ceil_div(K, BK);
  const long long pair_tiles = (long long)ceil_div(M, 256) * ceil_div(N, 256);
  if (tma && M > 128 && pair_tiles >= sms / 3) {
    p.pair = true;
    p.tile_m = p.tile_n = 256;
    p.tiles = pair_tiles;
    p.grid = 2 * pair_tiles;
    return p;
  }
  p.tile_n = BN;
  p.tile_m = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256;
  p.tiles = (long long)ceil_div(M, p.tile_m) * ceil_div(N, BN);
  const long long slots = (long long)sms * ctas_per_sm(p.tile_m);
  while (p.splits < 8 && p.tiles * p.splits * 2 <= slots && kb >= 4 * p.splits) p.splits *= 2;
  p.grid = p.tiles * p.splits;
  return p;
}

namespace {

template <int NT, int LOAD>
cudaError_t launch_stream(const CUtensorMap& tw, const CUtensorMap& ta, const StreamArgs& a, unsigned grid,
                          cudaStream_t s) {
  constexpr int ST = stages_for(NT);
  auto* kern = &i8_stream_kernel<NT, ST, LOAD>;
  static gpu::SmemOptIn optin;
  constexpr size_t smem = size_t(StreamLayout<NT, ST>::ALLOC);
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

template <int LOAD>
cudaError_t launch_stream(int nt, const CUtensorMap& tw, const CUtensorMap& ta, const StreamArgs& a, unsigned grid,
                          cudaStream_t s) {
  switch (nt) {
    case 16: return launch_stream<16, LOAD>(tw, ta, a, grid, s);
    case 32: return launch_stream<32, LOAD>(tw, ta, a, grid, s);
    case 64: return launch_stream<64, LOAD>(tw, ta, a, grid, s);
    case 128: return launch_stream<128, LOAD>(tw, ta, a, grid, s);
    default: return launch_stream<256, LOAD>(tw, ta, a, grid, s);
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
  cfg.blockDim = dim3(umma::kThreads);
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

}  // namespace

cudaError_t gemm(const Gemm& g, cudaStream_t s) {
  if (g.M == 0 || g.N == 0) return cudaSuccess;
  const gpu::Target* d = gpu::this_device();
  if (!d || d->cc != 100) return cudaErrorNotSupported;
  unsigned* status = nullptr;
  if (const cudaError_t e = status::word(&status); e != cudaSuccess) return e;
  bool tma = g.K > 0 && tma_rows(g.A, g.lda) && tma_rows(g.W, g.ldw);
  GemmPlan p = plan_gemm(g.M, g.N, g.K, tma, d->sms);
  CUtensorMap ta{}, tw{};
  if (tma && (!encode_map_i8(&ta, g.A, g.K, g.M, g.lda, p.pair ? 128 : p.tile_m) ||
              !encode_map_i8(&tw, g.W, g.K, g.N, g.ldw, 128))) {
    tma = false;  // the driver refused the geometry
    p = plan_gemm(g.M, g.N, g.K, false, d->sms);
  }
  if (p.pair) {
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
  StreamArgs a{};
  a.M = g.M;
  a.N = g.N;
  a.K = g.K;
  a.kb = ceil_div(g.K, BK);
  a.token_tiles = ceil_div(g.M, p.tile_m);
  a.splits = p.splits;
  a.weights_early = g.weights_settled;
  a.A = static_cast<const int8_t*>(g.A);
  a.W = static_cast<const int8_t*>(g.W);
  a.lda = g.lda;
  a.ldw = g.ldw;
  a.ldc = g.ldc;
  a.a_scale = g.a_scale;
  a.w_scale = g.w_scale;
  a.bias = g.bias;
  a.C = g.C;
  a.out = g.out;
  a.status = status;
  a.wait_limit_ns = kDefaultWaitLimitNs;
  return tma ? launch_stream<kLoadTma>(p.tile_m, tw, ta, a, unsigned(p.grid), s)
             : launch_stream<kLoadThreads>(p.tile_m, tw, ta, a, unsigned(p.grid), s);
}

}  // namespace aegis::i8
