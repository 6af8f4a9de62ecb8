// Pages (blocks) of a paged cache copied to other pages, in every plane of
// the allocation (K and V of every layer) by one launch: the copy on write of
// a forked sequence's last page, the moves of a compaction, a cache carried
// over into a smaller or larger one.
//
// Pure data movement, read once and written once: the gather's one-shot
// workgroups of 128 threads and 4 KiB (nkv_gather.hip), non-temporal, one
// per (piece of a page, pair, plane).  Bound by HBM: 2.7 GB read and written
// in 420 us, 6.5 TB/s; 63 copies of one page in 56 planes, written from the
// caches, 69 us at 6.6 TB/s; 7 pages in 2 planes 2.8 us, a launch's latency.
#include "nkv_common.h"

namespace nkv {
namespace {

constexpr int kCopyThreads = 128;
constexpr int kCopyBytes = 4096;  // per workgroup

template <int W>
__global__ __launch_bounds__(kCopyThreads) void copy_blocks_kernel(
    const uint8_t* __restrict__ src, uint8_t* __restrict__ dst, int64_t src_blocks, int64_t dst_blocks,
    int64_t block_bytes, int32_t pieces, const int2* __restrict__ pairs, int32_t num_pairs) {
  typedef typename Word<W>::type T;
  const int32_t pair = static_cast<int32_t>(blockIdx.x) / pieces;
  const int32_t piece = static_cast<int32_t>(blockIdx.x) - pair * pieces;
  const int2 p = pairs[pair];
  // Pairs outside the caches, or onto themselves, move nothing.
  if (p.x < 0 || p.x >= src_blocks || p.y < 0 || p.y >= dst_blocks || (src == dst && p.x == p.y)) return;
  const int64_t plane = blockIdx.y;
  const int64_t begin = static_cast<int64_t>(piece) * kCopyBytes;
  const int32_t words = static_cast<int32_t>(min(static_cast<int64_t>(kCopyBytes), block_bytes - begin) / W);
  const T* from = reinterpret_cast<const T*>(src + (plane * src_blocks + p.x) * block_bytes + begin);
  T* to = reinterpret_cast<T*>(dst + (plane * dst_blocks + p.y) * block_bytes + begin);
  // A page copied to several places (the samples of one prompt) is read
  // through the caches: its copies lie next to each other in the list.
  const bool again = (pair > 0 && pairs[pair - 1].x == p.x) || (pair + 1 < num_pairs && pairs[pair + 1].x == p.x);
  if (again) {
    for (int32_t w = threadIdx.x; w < words; w += kCopyThreads) store_stream(to + w, from[w]);
  } else {
    for (int32_t w = threadIdx.x; w < words; w += kCopyThreads) store_stream(to + w, load_stream(from + w));
  }
}

template <int W>
void launch_copy(dim3 grid, hipStream_t s, const void* src, void* dst, int64_t src_blocks,
                 int64_t dst_blocks, int64_t block_bytes, int32_t pieces, const int32_t* pairs,
                 int64_t num_pairs) {
  copy_blocks_kernel<W><<<grid, dim3(kCopyThreads), 0, s>>>(
      static_cast<const uint8_t*>(src), static_cast<uint8_t*>(dst), src_blocks, dst_blocks, block_bytes,
      pieces, reinterpret_cast<const int2*>(pairs), static_cast<int32_t>(num_pairs));
}

}  // namespace
}  // namespace nkv

extern "C" int nkv_copy_blocks(const void* src, void* dst, int64_t planes, int64_t src_blocks,
                               int64_t dst_blocks, int64_t block_bytes, const int32_t* pairs,
                               int64_t num_pairs, void* stream) {
  using namespace nkv;
  if (planes < 0 || src_blocks < 0 || dst_blocks < 0 || block_bytes <= 0 || num_pairs < 0 ||
      src_blocks > INT32_MAX || dst_blocks > INT32_MAX) {
    return nkv_fail(NKV_E_INVALID, "nkv_copy_blocks: negative or oversized planes, blocks or pairs");
  }
  if (planes == 0 || num_pairs == 0) return NKV_OK;
  if (!src || !dst || !pairs) return nkv_fail(NKV_E_INVALID, "nkv_copy_blocks: null pointer");
  if (reinterpret_cast<uint64_t>(pairs) % 8 != 0) {
    return nkv_fail(NKV_E_INVALID, "nkv_copy_blocks: pairs must be 8-byte aligned");
  }
  const int64_t pieces = (block_bytes + kCopyBytes - 1) / kCopyBytes;
  const int64_t most = UINT32_MAX / kCopyThreads;  // workgroups of a launch
  if (planes > 65535 || pieces > most || num_pairs > most / pieces) {
    return nkv_fail(NKV_E_INVALID, "nkv_copy_blocks: too many pages or planes for one launch");
  }
  const int w = common_word_bytes({reinterpret_cast<uint64_t>(src), reinterpret_cast<uint64_t>(dst),
                                   static_cast<uint64_t>(block_bytes)});
  const dim3 grid(static_cast<unsigned>(num_pairs * pieces), static_cast<unsigned>(planes));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto n = static_cast<int32_t>(pieces);
  switch (w) {
    case 16:
      launch_copy<16>(grid, s, src, dst, src_blocks, dst_blocks, block_bytes, n, pairs, num_pairs);
      break;
    case 8:
      launch_copy<8>(grid, s, src, dst, src_blocks, dst_blocks, block_bytes, n, pairs, num_pairs);
      break;
    case 4:
      launch_copy<4>(grid, s, src, dst, src_blocks, dst_blocks, block_bytes, n, pairs, num_pairs);
      break;
    case 2:
      launch_copy<2>(grid, s, src, dst, src_blocks, dst_blocks, block_bytes, n, pairs, num_pairs);
      break;
    default:
      return nkv_fail(NKV_E_INVALID, "nkv_copy_blocks: caches and pages must be 2-byte aligned");
  }
  return nkv_check_launch("nkv_copy_blocks");
}
