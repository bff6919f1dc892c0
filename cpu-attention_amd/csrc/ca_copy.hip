// Pages copied within the caches of several layers (copy_blocks): a pure copy, bytes as
// they are.
//
// One launch for every (array, pair, piece of a page): a block moves a piece of 16 KB, each
// thread 4 16-byte loads before any store.  The pages of a pair lie anywhere, so pieces
// are what keeps the reads long; the bytes are touched once (non-temporal).  A pair with
// a negative entry, with one past the cache, or of a page with itself moves nothing.
//
// Bound: reading and writing each page once (HBM).
#include "ca_device.h"
#include "ca_internal.h"

namespace ca {

constexpr int64_t kCopyPiece = 16384;

__global__ __launch_bounds__(256) void copy_kernel(CopyParams p) {
  const int64_t pieces = cdiv(p.bytes, kCopyPiece);
  const int64_t pair = blockIdx.x / pieces, at = (blockIdx.x - pair * pieces) * kCopyPiece;
  const int64_t src = p.mapping[2 * pair], dst = p.mapping[2 * pair + 1];
  if (src < 0 || dst < 0 || src >= p.nblocks || dst >= p.nblocks || src == dst) return;
  char* base = static_cast<char*>(p.base[blockIdx.y]);
  const char* from = base + src * p.bytes;
  char* to = base + dst * p.bytes;
  u32x4 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = at + (threadIdx.x + 256 * i) * 16;
    if (o < p.bytes) x[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + o));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = at + (threadIdx.x + 256 * i) * 16;
    if (o < p.bytes) __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4*>(to + o));
  }
}

// The rows of the 8-bit caches' scales: 4-byte words, one block of 64 per (array, pair).
__global__ __launch_bounds__(64) void copy_words_kernel(CopyParams p) {
  const int64_t src = p.mapping[2 * (int64_t)blockIdx.x], dst = p.mapping[2 * (int64_t)blockIdx.x + 1];
  if (src < 0 || dst < 0 || src >= p.nblocks || dst >= p.nblocks || src == dst) return;
  uint32_t* base = static_cast<uint32_t*>(p.base[blockIdx.y]);
  const int64_t words = p.bytes / 4;
  for (int64_t i = threadIdx.x; i < words; i += 64) base[dst * words + i] = base[src * words + i];
}

int copy_launch(const CopyParams& p, hipStream_t stream) {
  if (p.pairs == 0 || p.arrays == 0) return CA_OK;
  if (p.bytes % 16 == 0) {
    const int64_t gx = p.pairs * cdiv(p.bytes, kCopyPiece);
    if (gx > 0x7fffffff) return CA_DECLINED;
    hipLaunchKernelGGL(copy_kernel, dim3((unsigned)gx, (unsigned)p.arrays), dim3(256), 0, stream, p);
  } else {
    if (p.pairs > 0x7fffffff || p.bytes % 4) return CA_DECLINED;
    hipLaunchKernelGGL(copy_words_kernel, dim3((unsigned)p.pairs, (unsigned)p.arrays), dim3(64), 0, stream, p);
  }
  return ca_launch_status();
}

}  // namespace ca
