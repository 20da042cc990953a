// Copies of KV-cache pages: the first tokens[i] tokens of page src[i] to page dst[i],
// in every plane (layer, K or V) of the cache, in one launch.
//
// A copy has no arithmetic: its floor is each source token read once and each
// destination token written once.  Blocks take 16 KB pieces; the piece index
// varies slowest and the pair fastest, so the copies of one source page run side
// by side and all but the first read it from L2.
//
// The page lists are host data: they are checked here (range, a destination
// used twice, a destination that is also a source) and travel as kernel
// arguments, so there is no upload, no synchronisation and no buffer whose
// lifetime a captured graph would have to share.
#include "common.cuh"

#include <tuple>

namespace rlb {
namespace pages {

constexpr int kPairs = 640;     // pairs per launch
constexpr int kThreads = 256, kVec = 4;

struct Pairs {
  int src[kPairs], dst[kPairs], tokens[kPairs];
};

template <typename V>
__global__ void __launch_bounds__(kThreads)
copy_pages_kernel(const __grid_constant__ Pairs p, int n, uint8_t* __restrict__ cache, long long plane_bytes,
                  long long page_bytes, int token_bytes, int pieces) {
  constexpr long long kPiece = (long long)kThreads * kVec * sizeof(V);
  const long long i = blockIdx.x;
  const int pair = (int)(i % n);
  const int piece = (int)(i / n % pieces);
  const long long plane = i / n / pieces;
  const long long bytes = (long long)p.tokens[pair] * token_bytes;
  const long long o = piece * kPiece;
  if (o >= bytes) return;
  const uint8_t* s = cache + plane * plane_bytes + p.src[pair] * page_bytes + o;
  uint8_t* d = cache + plane * plane_bytes + p.dst[pair] * page_bytes + o;
  const int left = (int)(min(kPiece, bytes - o) / (long long)sizeof(V));
  V v[kVec];
#pragma unroll
  for (int k = 0; k < kVec; ++k)
    if (threadIdx.x + k * kThreads < left) v[k] = reinterpret_cast<const V*>(s)[threadIdx.x + k * kThreads];
#pragma unroll
  for (int k = 0; k < kVec; ++k)
    if (threadIdx.x + k * kThreads < left) reinterpret_cast<V*>(d)[threadIdx.x + k * kThreads] = v[k];
}

}  // namespace pages
}  // namespace rlb

using namespace rlb;

// cache [planes, pages, block, ...] contiguous, updated in place.  Returns (0, kernels launched), or what is
// wrong with the page lists and at which pair (nothing is copied then): 1 a page outside the cache,
// 2 a token count outside the page, 3 a page written twice, 4 a page both read and written.
std::tuple<int64_t, int64_t> copy_cache_pages(at::Tensor cache, std::vector<int64_t> src, std::vector<int64_t> dst,
                                              std::vector<int64_t> tokens) {
  RLB_CHECK(cache.is_cuda() && cache.dim() >= 3 && cache.is_contiguous(),
            "copy_cache_pages: a contiguous CUDA cache [planes, pages, block, ...] expected");
  RLB_CHECK(src.size() == dst.size() && src.size() == tokens.size(),
            "copy_cache_pages: src, dst and tokens must have one length");
  const int64_t planes = cache.size(0), pages = cache.size(1), block = cache.size(2);
  int64_t launches = 0;
  std::vector<uint8_t> written(src.empty() ? 0 : pages, 0);
  for (size_t i = 0; i < src.size(); ++i) {
    const int64_t at = i;
    if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages) return {1, at};
    if (tokens[i] < 0 || tokens[i] > block) return {2, at};
    if (written[dst[i]]) return {3, at};
    written[dst[i]] = 1;
  }
  for (size_t i = 0; i < src.size(); ++i)
    if (written[src[i]]) return {4, (int64_t)i};
  if (src.empty() || cache.numel() == 0) return {0, launches};
  const c10::cuda::CUDAGuard g(cache.device());
  const long long token_bytes = cache.numel() / (planes * pages * block) * cache.element_size();
  RLB_CHECK(token_bytes < (1 << 30), "copy_cache_pages: token too large");
  const long long page_bytes = token_bytes * block, plane_bytes = page_bytes * pages;
  const bool wide = token_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(cache.data_ptr()) % 16 == 0;
  const long long piece = (long long)pages::kThreads * pages::kVec * (wide ? 16 : 1);
  for (size_t i0 = 0; i0 < src.size(); i0 += pages::kPairs) {
    pages::Pairs p;
    const int n = (int)std::min<size_t>(pages::kPairs, src.size() - i0);
    int64_t most = 0;
    for (int i = 0; i < n; ++i) {
      p.src[i] = (int)src[i0 + i];
      p.dst[i] = (int)dst[i0 + i];
      p.tokens[i] = (int)tokens[i0 + i];
      most = std::max(most, tokens[i0 + i]);
    }
    if (most == 0) continue;
    const long long pieces = (most * token_bytes + piece - 1) / piece;
    const long long blocks = planes * pieces * n;
    RLB_CHECK(blocks < (1LL << 31) && pieces < (1LL << 31), "copy_cache_pages: too many bytes in one call");
    auto kern = wide ? pages::copy_pages_kernel<uint4> : pages::copy_pages_kernel<uint8_t>;
    kern<<<(unsigned)blocks, pages::kThreads, 0, stream()>>>(p, n, (uint8_t*)cache.data_ptr(), plane_bytes, page_bytes,
                                                             (int)token_bytes, (int)pieces);
    RLB_CUDA_CHECK(cudaGetLastError());
    ++launches;
  }
  return {0, launches};
}
