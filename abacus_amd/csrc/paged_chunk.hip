// The launch of a paged attention that may have chunks (paged_chunk.h) and single or drafted
// tokens (paged_few.h) beside each other: the chunks' blocks first, as they are the longest.
// In launches of their own the two took turns, and one that had nothing to do cost its
// 5 us: a chunk of 1000 tokens beside 24 single ones 60 us, together 47.
#include "paged_chunk.h"
#include "paged_few.h"

namespace abacus {
namespace {

template <bool Cd, int HD, bool Full, int QT>
__global__ __launch_bounds__(256, 2) void paged_both_kernel(PagedArgs few, PagedArgs many, int many_blocks) {
  constexpr size_t kBytes = sizeof(ChunkLds<HD>) > sizeof(FewLds<HD, QT>) ? sizeof(ChunkLds<HD>) : sizeof(FewLds<HD, QT>);
  __shared__ __attribute__((aligned(1024))) char lds[kBytes];
  if ((int)blockIdx.x < many_blocks) {
    chunk_block<Cd, HD, Full>(many, blockIdx.x, *reinterpret_cast<ChunkLds<HD>*>(lds));
  } else {
    few_block<uint16_t, Cd, HD, Full, QT>(few, (int)blockIdx.x - many_blocks, (int)gridDim.x - many_blocks,
                                          *reinterpret_cast<FewLds<HD, QT>*>(lds));
  }
}

template <bool Cd, int QT>
void launch_both_of(const PagedArgs& few, const PagedArgs& many, unsigned blocks, int many_blocks, hipStream_t s) {
  const dim3 grid(blocks), threads(256);
  if (few.K == 64) hipLaunchKernelGGL((paged_both_kernel<Cd, 64, true, QT>), grid, threads, 0, s, few, many, many_blocks);
  else if (few.K == 128) hipLaunchKernelGGL((paged_both_kernel<Cd, 128, true, QT>), grid, threads, 0, s, few, many, many_blocks);
  else if (few.K < 64) hipLaunchKernelGGL((paged_both_kernel<Cd, 64, false, QT>), grid, threads, 0, s, few, many, many_blocks);
  else hipLaunchKernelGGL((paged_both_kernel<Cd, 128, false, QT>), grid, threads, 0, s, few, many, many_blocks);
}

}  // namespace

int launch_both(const PagedArgs& few, const PagedArgs& many, unsigned few_blocks, unsigned many_blocks, int few_rows,
                bool codes, hipStream_t s) {
  const unsigned blocks = few_blocks + many_blocks;
  const int m = (int)many_blocks;
  if (few_rows == 16) codes ? launch_both_of<true, 1>(few, many, blocks, m, s) : launch_both_of<false, 1>(few, many, blocks, m, s);
  else codes ? launch_both_of<true, 2>(few, many, blocks, m, s) : launch_both_of<false, 2>(few, many, blocks, m, s);
  ABACUS_CHECK_LAUNCH("paged_attention (chunk)");
  return 0;
}

}  // namespace abacus
