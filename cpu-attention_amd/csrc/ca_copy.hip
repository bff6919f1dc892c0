// Pages copied within the caches of several layers (copy_blocks): a pure copy, bytes as
// they are.
//
// One launch for every (array, pair, piece of a page), up to kCopyArrays arrays: a block
// moves a piece of 16 KB, each thread 4 16-byte loads before any store.  The pages of a
// pair lie anywhere, so pieces are what keeps the reads long; the bytes are touched once
// (non-temporal).  An 8-bit cache's scales are arrays of their own in the same launch,
// whose rows of 4-byte words the first piece's block moves.  A pair with a negative entry,
// with one past the cache, or of a page with itself moves nothing.
//
// Bound: reading and writing each page once (HBM); the launch for a few pages.
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
  if ((int)blockIdx.y >= p.caches) {
    if (at != 0) return;
    const uint32_t* from = reinterpret_cast<const uint32_t*>(base + src * p.row_bytes);
    uint32_t* to = reinterpret_cast<uint32_t*>(base + dst * p.row_bytes);
    for (int64_t i = threadIdx.x; i < p.row_bytes / 4; i += 256) to[i] = from[i];
    return;
  }
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

int copy_launch(const CopyParams& p, hipStream_t stream) {
  if (p.pairs == 0 || p.arrays == 0) return CA_OK;
  const int64_t gx = p.pairs * cdiv(p.bytes, kCopyPiece);
  if (gx > 0x7fffffff) return CA_DECLINED;
  hipLaunchKernelGGL(copy_kernel, dim3((unsigned)gx, (unsigned)p.arrays), dim3(256), 0, stream, p);
  return ca_launch_status();
}

}  // namespace ca
