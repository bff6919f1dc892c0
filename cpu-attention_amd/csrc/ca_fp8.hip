// Tokens into the 8-bit cache: e4m3 codes with one power-of-two scale per (page, head),
// for K and for V each.
//
// The rule and a page's store are ca_fp8.h's (store_page).
//
// Work split: one wave per (page, head).  It reads the head's rows of the page's tokens
// (16 positions at a time, 8 dims per lane: the next positions' loads are all in flight),
// takes both maxima by a wave reduction, rescales if it must, and writes V's rows as they
// come and K's words transposed through LDS, 16 bytes (4 neighbouring tokens) at a time.
// Nobody else touches the page's codes or scales, so nothing is atomic and the result
// does not depend on the order of anything.
//
// Which tokens a page gets:
//   append mode  (decode): positions lens[s] .. + per_seq - 1 of sequence s, by arithmetic;
//   slot mode    (reshape_and_cache_fp8): slots in any order, of many pages.  A slot named
//                twice takes its last token.  Up to kScanTokens tokens, each wave's block
//                scans the slots for its page's (the block of a page's first token does the
//                page).  Above, two kernels write each slot's last token into a table over
//                the cache's slots and list the pages, and a fixed grid walks that list.
//
// Bound: reading the tokens and writing their codes (HBM); launches for a few tokens.
#include "ca_device.h"
#include "ca_fp8.h"
#include "ca_internal.h"

namespace ca {

constexpr int kStore8Waves = 4;       // heads per block
// Blocks that walk the listed pages: one unit each up to here (128 prompts of 64 to 1024
// tokens, H=32 E=128, 35000 units: 4096 blocks 442 us, 16384 425, 65536 420, more the same).
constexpr int64_t kStore8Grid = 65536;
// Tokens up to which each block scans the slots (scan / list, E=128 page 16: 256 tokens H=8
// 6.5 / 10.4 us, H=32 10.0 / 11.2; 512 8.9 / 10.7 and 13.6 / 12.3; 1024 16.3 / 11.0 and 25.3 /
// 13.7).
constexpr int64_t kScanTokens = 512;
constexpr int64_t kScanPage = 1024;    // positions of a page up to which it can

// Append mode: block (sequence and 4 heads, k-th page from position lens[s] on).
template <int E, bool BF>
__global__ __launch_bounds__(64 * kStore8Waves) void store8_append_kernel(Store8Params p) {
  __shared__ __attribute__((aligned(16))) uint32_t kl[kStore8Waves][Store8Shape<E>::LDS_WORDS];
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t hg = cdiv(p.heads, kStore8Waves);
  const int64_t seq = blockIdx.x / hg, h = (blockIdx.x - seq * hg) * kStore8Waves + wv;
  if (h >= p.heads) return;
  const int64_t len = p.lens[seq], n = p.per_seq;
  if (len < 0) return;
  for (int64_t pi = len / p.page + blockIdx.y; pi < p.pt_width && pi * p.page < len + n; pi += gridDim.y) {
    const int64_t blk = p.page_table[seq * p.pt_width + pi], first = pi * p.page;
    if (blk < 0 || blk >= p.nblocks) continue;
    store_page<E, BF>(p, blk, h, kl[wv], [&](int64_t t) -> int {
      const int64_t i = first + t - len;
      return i >= 0 && i < n ? (int)(seq * n + i) : -1;
    });
  }
}

// The page of slot s, or -1 for padding and slots past the cache.
__device__ __forceinline__ int64_t slot_page(const Store8Params& p, int64_t s) {
  return s >= 0 && s < p.nblocks * p.page ? s / p.page : -1;
}

// Slot mode, few tokens: block (token, 4 heads); the block of a page's first token does
// the page.
template <int E, bool BF>
__global__ __launch_bounds__(64 * kStore8Waves) void store8_scan_kernel(Store8Params p) {
  __shared__ __attribute__((aligned(16))) uint32_t kl[kStore8Waves][Store8Shape<E>::LDS_WORDS];
  __shared__ int owner[kScanPage];
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t hg = cdiv(p.heads, kStore8Waves);
  const int64_t i = blockIdx.x / hg, h = (blockIdx.x - i * hg) * kStore8Waves + wv;
  const int64_t blk = slot_page(p, p.slots[i]);
  if (blk < 0) return;
  for (int t = threadIdx.x; t < p.page; t += 64 * kStore8Waves) owner[t] = -1;
  __syncthreads();
  bool earlier = false;
  for (int64_t j = threadIdx.x; j < p.ntok; j += 64 * kStore8Waves) {
    const uint64_t t = (uint64_t)p.slots[j] - (uint64_t)(blk * p.page);
    if (t < (uint64_t)p.page) {
      earlier |= j < i;
      atomicMax(&owner[t], (int)j);
    }
  }
  if (__syncthreads_or(earlier) || h >= p.heads) return;
  store_page<E, BF>(p, blk, h, kl[wv], [&](int64_t t) -> int { return owner[t]; });
}

// Slot mode, many tokens.  p.work: [slots of the cache] each slot's last token, [blocks]
// whether a page is listed, the number of pages listed, the pages; all -1 at first (the
// number counts from -1).
__device__ __forceinline__ int32_t* work_listed(const Store8Params& p) { return p.work + p.nblocks * p.page; }
__device__ __forceinline__ int32_t* work_count(const Store8Params& p) { return work_listed(p) + p.nblocks; }

__global__ __launch_bounds__(256) void store8_clear_kernel(int32_t* work, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) work[i] = -1;
}

// A block's pages are counted in LDS first: one addition to the common number per block
// (one per page took 16.8 us for 65536 tokens on 4400 pages, this 6.6).
__global__ __launch_bounds__(256) void store8_list_kernel(Store8Params p) {
  __shared__ int pages, base;
  if (threadIdx.x == 0) pages = 0;
  __syncthreads();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t blk = -1;
  int at = -1;
  if (i < p.ntok) {
    const int64_t s = p.slots[i];
    blk = slot_page(p, s);
    if (blk >= 0) {
      atomicMax(p.work + s, (int)i);
      // A run of tokens of one page asks once.
      if ((i == 0 || slot_page(p, p.slots[i - 1]) != blk) && atomicExch(work_listed(p) + blk, 0) == -1)
        at = atomicAdd(&pages, 1);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && pages > 0) base = atomicAdd(work_count(p), pages);
  __syncthreads();
  if (at >= 0) work_count(p)[2 + base + at] = (int)blk;
}

template <int E, bool BF>
__global__ __launch_bounds__(64 * kStore8Waves) __attribute__((amdgpu_waves_per_eu(4))) void store8_pages_kernel(Store8Params p) {
  __shared__ __attribute__((aligned(16))) uint32_t kl[kStore8Waves][Store8Shape<E>::LDS_WORDS];
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t hg = cdiv(p.heads, kStore8Waves);
  const int32_t* count = work_count(p);
  const int64_t units = ((int64_t)count[0] + 1) * hg;
  for (int64_t i0 = blockIdx.x; i0 < units; i0 += gridDim.x) {
    const int64_t u = xcd_remap(i0, units);  // a page's heads on one XCD: they read the same rows
    const int64_t i = u / hg, h = (u - i * hg) * kStore8Waves + wv;
    if (h >= p.heads) continue;
    const int64_t blk = count[1 + i];
    const int32_t* owner = p.work + blk * p.page;
    store_page<E, BF>(p, blk, h, kl[wv], [&](int64_t t) -> int { return owner[t]; });
  }
}

int64_t store8_work_ints(int64_t ntok, int64_t nblocks, int64_t page) {
  if (ntok <= kScanTokens && page <= kScanPage) return 0;
  return nblocks * page + nblocks + 1 + (ntok < nblocks ? ntok : nblocks);
}

template <int E, bool BF>
static int store8_launch_t(const Store8Params& p, hipStream_t stream) {
  const int64_t hg = cdiv(p.heads, kStore8Waves);
  const dim3 block(64 * kStore8Waves);
  if (p.ntok > 0x7fffffff) return CA_DECLINED;
  if (!p.slots) {
    const int64_t gx = p.ntok / p.per_seq * hg, gy = (p.per_seq + p.page - 2) / p.page + 1;  // pages of per_seq tokens
    if (gx > 0x7fffffff) return CA_DECLINED;
    hipLaunchKernelGGL((store8_append_kernel<E, BF>), dim3((unsigned)gx, (unsigned)(gy < 65535 ? gy : 65535)), block, 0, stream, p);
    return ca_launch_status();
  }
  if (p.nblocks > 0x7fffffff) return CA_DECLINED;
  const int64_t ints = store8_work_ints(p.ntok, p.nblocks, p.page);
  if (ints == 0) {
    if (p.ntok * hg > 0x7fffffff) return CA_DECLINED;
    hipLaunchKernelGGL((store8_scan_kernel<E, BF>), dim3((unsigned)(p.ntok * hg)), block, 0, stream, p);
    return ca_launch_status();
  }
  const int64_t cb = cdiv(ints, 1024);
  hipLaunchKernelGGL(store8_clear_kernel, dim3((unsigned)(cb < 4096 ? cb : 4096)), dim3(256), 0, stream, p.work, ints);
  int st = ca_launch_status();
  if (st != CA_OK) return st;
  hipLaunchKernelGGL(store8_list_kernel, dim3((unsigned)cdiv(p.ntok, 256)), dim3(256), 0, stream, p);
  st = ca_launch_status();
  if (st != CA_OK) return st;
  const int64_t most = (p.ntok < p.nblocks ? p.ntok : p.nblocks) * hg;
  hipLaunchKernelGGL((store8_pages_kernel<E, BF>), dim3((unsigned)(most < kStore8Grid ? most : kStore8Grid)), block, 0, stream, p);
  return ca_launch_status();
}

template <bool BF>
static int store8_launch_e(const Store8Params& p, int E, hipStream_t stream) {
  switch (E) {
    case 32: return store8_launch_t<32, BF>(p, stream);
    case 64: return store8_launch_t<64, BF>(p, stream);
    case 128: return store8_launch_t<128, BF>(p, stream);
  }
  return CA_DECLINED;
}

int store8_launch(const Store8Params& p, int E, int bf16, hipStream_t stream) {
  if (p.ntok == 0) return CA_OK;
  return bf16 ? store8_launch_e<true>(p, E, stream) : store8_launch_e<false>(p, E, stream);
}

}  // namespace ca
