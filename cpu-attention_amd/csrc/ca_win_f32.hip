// fp32 prefill with a sliding window and sinks, in 32-bit MFMAs.
//
// Semantics as the bf16 window kernel (ca_duo.h): win_tiles lists a block's keys, the
// rows' own limits are masked in the tiles, the softmax runs in base 2 with a running
// max, P and all sums are fp32, a row that sees no key is exactly 0, and rows that come
// out not finite are redone key by key (win_redo_row).
//
// S^T = K Q^T and O^T += V^T P^T in 32x32x2 MFMAs: a lane owns one query row (li) and 16
// of a tile's 32 keys, whose probabilities are the B operand of P.V as they stand.  K and V
// tiles go global -> registers -> LDS, the next tile's loads in flight during a tile.
//
// A block is 4 waves.  KW = 1: 32 rows each (128 per block), sharing 32-key tiles.  KW = 4:
// the same 32 rows, each wave 32 of a tile's 128 keys, merged in LDS at the end: four times
// the blocks of a quarter of the walk, for calls whose 128-row blocks leave CUs idle.
//
// Bound: the 32-bit MFMAs (157 TFLOP/s dense); masked parts of the window's edge tiles are
// computed too.
#include <type_traits>

#include "ca_device.h"
#include "ca_internal.h"
#include "ca_window.h"

namespace ca {

template <int E, int KW>
struct WinF32Cfg {
  static constexpr int BM = 128 / KW;       // rows per block
  static constexpr int BN = 32 * KW;        // keys per tile
  static constexpr int KS = E + 2;          // K row stride (floats): conflict-free 8-byte reads
  static constexpr int CH = BN * E / 1024;  // 16-byte chunks per thread (K and V each)
  static constexpr int V0 = BN * KS;        // V after K (floats)
  static constexpr int MERGE = 32 * E + 128;  // a wave's O, m and l for the merge (floats)
  static constexpr int TILES = BN * (KS + E);
  static constexpr int LDS_BYTES = 4 * (KW > 1 && 4 * MERGE > TILES ? 4 * MERGE : TILES);
  static_assert(CH * 1024 == BN * E && V0 % 4 == 0, "tile shape");
};

template <int E, int KW>
__global__ __launch_bounds__(256, KW == 1 ? 2 : 1) void win_f32_kernel(WindowParams p) {
  using C = WinF32Cfg<E, KW>;
  constexpr int BM = C::BM, BN = C::BN, KS = C::KS, CH = C::CH, ND = E / 32;
  extern __shared__ __attribute__((aligned(16))) float win_smem[];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 31, hf = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = KW == 1 ? 0 : wv, rw = KW == 1 ? wv : 0;
  const int L = (int)p.seq_q, S = (int)p.seq_k, diag = S - L;
  const int nqb = (L + BM - 1) / BM;
  const int64_t lg = xcd_remap(blockIdx.x, gridDim.x), bh = lg / nqb, b = bh / p.heads, h = bh - b * p.heads;
  const int q0 = (nqb - 1 - (int)(lg - bh * nqb)) * BM, r0 = q0 + 32 * rw, row = r0 + li;
  const uint32_t* qg = reinterpret_cast<const uint32_t*>(p.q) + b * p.qs[0] + h * p.qs[2];
  const uint32_t* kg = reinterpret_cast<const uint32_t*>(p.k) + b * p.ks[0] + h * p.ks[2];
  const uint32_t* vg = reinterpret_cast<const uint32_t*>(p.v) + b * p.vs[0] + h * p.vs[2];
  const WinTiles wt = win_tiles(p, q0, BM, BN);

  // Q: lane (row li, half hf) holds dims 4t + 2hf and 4t + 2hf + 1.
  float qr[E / 2];
#pragma unroll
  for (int t = 0; t < E / 4; ++t) {
    u32x2 x = {0, 0};
    if (row < L) x = *reinterpret_cast<const u32x2*>(qg + (int64_t)row * p.qs[1] + 4 * t + 2 * hf);
    qr[2 * t] = __uint_as_float(x.x);
    qr[2 * t + 1] = __uint_as_float(x.y);
  }

  // Chunk i of thread tid: key (tid + 256 i) / (E / 4) of the tile, dims 4 ((tid + 256 i) % (E / 4)).
  u32x4 kreg[CH], vreg[CH];
  auto load_tile = [&](int t) {
    const int k0 = win_key0(wt, t, BN);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + 256 * i, r = c / (E / 4), c4 = c % (E / 4);
      const int64_t key = k0 + r;
      kreg[i] = vreg[i] = u32x4{0, 0, 0, 0};
      if (t < wt.n && key < S) {
        kreg[i] = *reinterpret_cast<const u32x4*>(kg + key * p.ks[1] + 4 * c4);
        vreg[i] = *reinterpret_cast<const u32x4*>(vg + key * p.vs[1] + 4 * c4);
      }
    }
  };
  auto store_tile = [&]() {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + 256 * i, r = c / (E / 4), c4 = c % (E / 4);
      uint32_t* kd = reinterpret_cast<uint32_t*>(win_smem) + r * KS + 4 * c4;
      *reinterpret_cast<u32x2*>(kd) = u32x2{kreg[i].x, kreg[i].y};
      *reinterpret_cast<u32x2*>(kd + 2) = u32x2{kreg[i].z, kreg[i].w};
      *reinterpret_cast<u32x4*>(win_smem + C::V0 + r * E + 4 * c4) = vreg[i];
    }
  };

  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x16{};
  float m = -INFINITY, l = 0.f;
  const float* kb = win_smem + 32 * kw * KS;
  const float* vb = win_smem + C::V0 + 32 * kw * E;
  const int rhi = imin(S - 1, row + diag + p.right), rlo = imax(0, row + diag - p.left);
  load_tile(0);
  for (int t = 0; t < wt.n; ++t) {
    store_tile();
    __syncthreads();
    load_tile(t + 1);
    const int k0 = win_key0(wt, t, BN) + 32 * kw, pos = r0 + diag;  // this wave's keys; its first row's position
    if (r0 < L && k0 < S && k0 <= pos + 31 + p.right && (k0 + 31 >= pos - p.left || k0 < p.sinks)) {
      f32x16 st = f32x16{};
#pragma unroll
      for (int t4 = 0; t4 < E / 4; ++t4) {
        const u32x2 a = *reinterpret_cast<const u32x2*>(kb + li * KS + 4 * t4 + 2 * hf);
        st = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), qr[2 * t4], st, 0, 0, 0);
        st = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), qr[2 * t4 + 1], st, 0, 0, 0);
      }
      const int hi = rhi - k0 - 4 * hf, lo = rlo - k0 - 4 * hf, sk = p.sinks - k0 - 4 * hf;
      const bool all = k0 + 32 <= imin(S, pos + p.right + 1) && (k0 >= pos + 31 - p.left || k0 + 32 <= p.sinks);
      float x[16], mt = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = 8 * (r >> 2) + (r & 3);
        x[r] = all || (j <= hi && (j >= lo || j < sk)) ? st[r] * p.c : -INFINITY;
        mt = fmaxf(mt, x[r]);
      }
      const float mn = fmaxf(m, fmaxf(mt, __shfl_xor(mt, 32))), mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - mu);
      m = mn;
      float ls = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[r] = __builtin_amdgcn_exp2f(x[r] - mu);
        ls += x[r];
      }
      l = l * alpha + ls;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= alpha;
      // O^T += V^T P^T, two keys per step: step r takes keys 8 (r / 4) + 4 hf + r % 4.
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = 8 * (r >> 2) + 4 * hf + (r & 3);
#pragma unroll
        for (int d = 0; d < ND; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vb[key * E + 32 * d + li], x[r], o[d], 0, 0, 0);
      }
    }
    __syncthreads();
  }

  if constexpr (KW > 1) {
    float* mb = win_smem + wv * C::MERGE + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) mb[64 * (16 * d + r)] = o[d][r];
    mb[32 * E] = m;
    mb[32 * E + 64] = l;
    __syncthreads();
    if (wv != 0) return;
#pragma unroll
    for (int w = 1; w < KW; ++w) {
      const float* ob = win_smem + w * C::MERGE + lane;
      const float m1 = ob[32 * E], mn = fmaxf(m, m1), mu = mn == -INFINITY ? 0.f : mn;
      const float w0 = __builtin_amdgcn_exp2f(m - mu), w1 = __builtin_amdgcn_exp2f(m1 - mu);
      m = mn;
      l = l * w0 + ob[32 * E + 64] * w1;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * w0 + ob[64 * (16 * d + r)] * w1;
    }
  }
  const float lt = l + __shfl_xor(l, 32), inv = lt > 0.f ? 1.f / lt : 0.f;
  float* out = reinterpret_cast<float*>(p.out) + (b * p.seq_q * p.heads + h) * E;
  bool bad = !(fabsf(lt) < INFINITY);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bad |= !(fabsf(o[d][4 * g + j]) < INFINITY);
        x[j] = o[d][4 * g + j] * inv;
      }
      if (row < L) *reinterpret_cast<f32x4*>(out + (int64_t)row * p.heads * E + 32 * d + 8 * g + 4 * hf) = x;
    }
  const uint64_t bits = __ballot(bad);
  uint32_t redo = (uint32_t)bits | (uint32_t)(bits >> 32);
  if (__builtin_expect(redo == 0, 1)) return;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  while (redo) {
    const int r = r0 + __builtin_ctz(redo);
    redo &= redo - 1;
    if (r >= L) continue;
    win_redo_row<E, uint32_t, BN>(p, wt, 0, wt.n, qg, kg, vg, r, [&](float rm, float rl, int d, float a) {
      out[(int64_t)r * p.heads * E + d] = rl != 0.f ? a / rl : 0.f;
    });
  }
}

template <int E, int KW>
static int win_f32_launch_t(const WindowParams& p, hipStream_t stream) {
  using C = WinF32Cfg<E, KW>;
  const int64_t nb = p.batch * p.heads * cdiv(p.seq_q, C::BM);
  if (nb > 0x7fffffff) return CA_DECLINED;
  if (C::LDS_BYTES > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(win_f32_kernel<E, KW>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS_BYTES);
    if (e != hipSuccess) return CA_HIP_ERROR - (int)e;
  }
  hipLaunchKernelGGL((win_f32_kernel<E, KW>), dim3((unsigned)nb), dim3(256), C::LDS_BYTES, stream, p);
  return ca_launch_status();
}

template <int E>
static int win_f32_launch_e(const WindowParams& p, hipStream_t stream) {
  return p.batch * p.heads * cdiv(p.seq_q, 128) <= 256 ? win_f32_launch_t<E, 4>(p, stream) : win_f32_launch_t<E, 1>(p, stream);
}

int flash_window_f32_launch(const WindowParams& p, int E, hipStream_t stream) {
  if (!window_fits(p, E, 4)) return CA_DECLINED;
  switch (E) {
    case 32: return win_f32_launch_e<32>(p, stream);
    case 64: return win_f32_launch_e<64>(p, stream);
    case 128: return win_f32_launch_e<128>(p, stream);
  }
  return CA_DECLINED;
}

}  // namespace ca
