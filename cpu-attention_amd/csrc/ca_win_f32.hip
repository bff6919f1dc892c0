// fp32 prefill with a sliding window and sinks, in 32-bit MFMAs.
//
// Semantics as the bf16 window kernel (ca_duo.h): win_tiles lists a block's keys, the
// rows' own limits are masked in the tiles, the softmax runs in base 2 with a running
// max, P and all sums are fp32, a row that sees no key is exactly 0, and rows that come
// out not finite are redone key by key (win_redo_row).
//
// S^T = K Q^T and O^T += V^T P^T in 32-bit MFMAs of RB = 32 rows (32x32x2) or 16 (16x16x4):
// lane l owns query row l % RB and, of every RB keys, those whose probabilities are its B
// operand of P.V as they stand.  K and V tiles go global -> registers -> LDS, the next
// tile's loads in flight during a tile.
//
// A block is 4 waves.  KW = 1: 32 rows each (128 per block), sharing 32-key tiles.  KW = 4:
// the same RB rows, each wave 32 of a tile's 128 keys, merged in LDS at the end: for calls
// whose 128-row blocks leave CUs idle, four or (RB = 16) eight times the blocks.
//
// SPLIT: few rows over long windows; blockIdx.y takes a share of the tiles and leaves its
// rows' partials (O, max, sum) for the combine kernel.
//
// Runs calls of few rows or few visible keys (flash_window_f32_blocks in ca_flash.hip says
// which run on split operands) and, with p.redo, the 128-row blocks of the others whose
// values those do not hold.
//
// Bound: the 32-bit MFMAs (157 TFLOP/s dense), either shape; masked parts of the window's
// edge tiles are computed too.
#include <type_traits>

#include "ca_device.h"
#include "ca_internal.h"
#include "ca_window.h"

namespace ca {

template <int E, int KW, int RB>
struct WinF32Cfg {
  static constexpr int BM = 4 * RB / KW;    // rows per block
  static constexpr int BN = 32 * KW;        // keys per tile
  static constexpr int RS = E + 4;          // K and V row stride (floats): conflict-free operand reads
  static constexpr int CH = BN * E / 1024;  // 16-byte chunks per thread (K and V each)
  static constexpr int NO = RB * E / 64;    // O registers per lane
  static constexpr int MERGE = 64 * (NO + 2);  // a wave's O, m and l for the merge (floats)
  static constexpr int TILES = 2 * BN * RS;
  static constexpr int LDS_BYTES = 4 * (KW > 1 && 4 * MERGE > TILES ? 4 * MERGE : TILES);
  static_assert(CH * 1024 == BN * E, "tile shape");
};

template <int E, int KW, int RB, bool SPLIT>
__global__ __launch_bounds__(256, KW == 1 ? 2 : 1) void win_f32_kernel(WindowParams p) {
  using C = WinF32Cfg<E, KW, RB>;
  constexpr int BM = C::BM, BN = C::BN, RS = C::RS, CH = C::CH, NO = C::NO;
  constexpr int NQ = 64 / RB;       // lanes per row (lane quarter or half qd)
  constexpr int NB = 32 / RB;       // RB-key blocks of a wave's 32 keys
  constexpr int NS = RB * RB / 64;  // accumulator registers of an RB x RB block
  constexpr int ND = E / RB;        // RB-dim blocks of O
  typedef __attribute__((ext_vector_type(NS))) float acc_t;
  extern __shared__ __attribute__((aligned(16))) float win_smem[];
  const int tid = threadIdx.x, lane = tid & 63, li = lane % RB, qd = lane / RB;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = KW == 1 ? 0 : wv, rw = KW == 1 ? wv : 0;
  const int L = (int)p.seq_q, S = (int)p.seq_k, diag = S - L;
  const uint32_t nqb = (uint32_t)(L + BM - 1) / BM, heads = (uint32_t)p.heads;
  const uint32_t lg = (uint32_t)xcd_remap(blockIdx.x, gridDim.x), bh = lg / nqb, bi = bh / heads;
  const int64_t b = bi, h = bh - bi * heads;
  const int q0 = (int)(nqb - 1 - (lg - bh * nqb)) * BM, r0 = q0 + RB * rw, row = r0 + li;
  const uint32_t* qg = reinterpret_cast<const uint32_t*>(p.q) + b * p.qs[0] + h * p.qs[2];
  const uint32_t* kg = reinterpret_cast<const uint32_t*>(p.k) + b * p.ks[0] + h * p.ks[2];
  const uint32_t* vg = reinterpret_cast<const uint32_t*>(p.v) + b * p.vs[0] + h * p.vs[2];
  if (KW == 1 && p.redo && !p.redo[((int64_t)bh * nqb + q0 / BM) * gridDim.y + blockIdx.y]) return;
  const WinTiles wt = win_tiles(p, q0, BM, BN);
  // The block's tiles [t0, t1) of the list.
  const int share = SPLIT ? (wt.n + (int)gridDim.y - 1) / (int)gridDim.y : wt.n;
  const int t0 = SPLIT ? imin((int)blockIdx.y * share, wt.n) : 0, t1 = imin(t0 + share, wt.n);

  // Chunk i of thread tid: key (tid + 256 i) / (E / 4) of the tile, dims 4 ((tid + 256 i) % (E / 4)).
  u32x4 kreg[CH], vreg[CH];
  auto load_tile = [&](int t) {
    const int k0 = win_key0(wt, t, BN);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + 256 * i, r = c / (E / 4), c4 = c % (E / 4);
      const int64_t key = k0 + r;
      kreg[i] = vreg[i] = u32x4{0, 0, 0, 0};
      if (t < t1 && key < S) {
        kreg[i] = *reinterpret_cast<const u32x4*>(kg + key * p.ks[1] + 4 * c4);
        vreg[i] = *reinterpret_cast<const u32x4*>(vg + key * p.vs[1] + 4 * c4);
      }
    }
  };
  auto store_tile = [&]() {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + 256 * i, r = c / (E / 4), c4 = c % (E / 4);
      *reinterpret_cast<u32x4*>(win_smem + r * RS + 4 * c4) = kreg[i];
      *reinterpret_cast<u32x4*>(win_smem + (BN + r) * RS + 4 * c4) = vreg[i];
    }
  };
  load_tile(t0);

  // Q: the lane's row, dims 4 NQ u + 4 qd + e in qr[4 u + e]: the dims that MFMA step 4 u + e
  // takes of each lane, of K's rows too.
  float qr[E / NQ];
#pragma unroll
  for (int u = 0; u < E / (4 * NQ); ++u) {
    u32x4 x = {0, 0, 0, 0};
    if (row < L) x = *reinterpret_cast<const u32x4*>(qg + (int64_t)row * p.qs[1] + 4 * NQ * u + 4 * qd);
#pragma unroll
    for (int e = 0; e < 4; ++e) qr[4 * u + e] = __uint_as_float(x[e]);
  }
  auto mfma = [](float a, float bb, acc_t c) __attribute__((always_inline)) {
    if constexpr (RB == 32) return __builtin_amdgcn_mfma_f32_32x32x2f32(a, bb, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x4f32(a, bb, c, 0, 0, 0);
  };

  acc_t o[ND];  // O^T: dims RB d + acc_row(r)
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = acc_t{};
  float m = -INFINITY, l = 0.f;
  const float* kb = win_smem + 32 * kw * RS;
  const float* vb = win_smem + (BN + 32 * kw) * RS;
  // Row of an RB x RB block that register r of the lane holds (its column is li), less 4 qd.
  auto acc_row = [](int r) { return 4 * NQ * (r >> 2) + (r & 3); };
  const int rhi = imin(S - 1, row + diag + p.right), rlo = imax(0, row + diag - p.left);
  for (int t = t0; t < t1; ++t) {
    store_tile();
    __syncthreads();
    load_tile(t + 1);
    const int k0 = win_key0(wt, t, BN) + 32 * kw, pos = r0 + diag;  // this wave's keys; its first row's position
    if (r0 < L && k0 < S && k0 <= pos + RB - 1 + p.right && (k0 + 31 >= pos - p.left || k0 < p.sinks)) {
      acc_t st[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        st[n] = acc_t{};
#pragma unroll
        for (int u = 0; u < E / (4 * NQ); ++u) {
          const f32x4 a = *reinterpret_cast<const f32x4*>(kb + (RB * n + li) * RS + 4 * NQ * u + 4 * qd);
#pragma unroll
          for (int e = 0; e < 4; ++e) st[n] = mfma(a[e], qr[4 * u + e], st[n]);
        }
      }
      const int hi = rhi - k0 - 4 * qd, lo = rlo - k0 - 4 * qd, sk = p.sinks - k0 - 4 * qd;
      const bool all = k0 + 32 <= imin(S, pos + p.right + 1) && (k0 >= pos + RB - 1 - p.left || k0 + 32 <= p.sinks);
      float x[NB][NS], mt = -INFINITY;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < NS; ++r) {
          const int j = RB * n + acc_row(r);
          x[n][r] = all | ((j <= hi) & ((j >= lo) | (j < sk))) ? st[n][r] * p.c : -INFINITY;  // (no branches)
          mt = fmaxf(mt, x[n][r]);
        }
#pragma unroll
      for (int w = RB; w < 64; w <<= 1) mt = fmaxf(mt, __shfl_xor(mt, w));
      const float mn = fmaxf(m, mt), mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - mu);
      m = mn;
      float ls = 0.f;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < NS; ++r) {
          x[n][r] = __builtin_amdgcn_exp2f(x[n][r] - mu);
          ls += x[n][r];
        }
      l = l * alpha + ls;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= alpha;
      // O^T += V^T P^T: step r takes of each lane the key whose probability it holds there.
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < NS; ++r) {
          const float* vr = vb + (RB * n + acc_row(r) + 4 * qd) * RS + li;
#pragma unroll
          for (int d = 0; d < ND; ++d) o[d] = mfma(vr[RB * d], x[n][r], o[d]);
        }
    }
    __syncthreads();
  }

  if constexpr (KW > 1) {
    float* mb = win_smem + wv * C::MERGE + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < NS; ++r) mb[64 * (NS * d + r)] = o[d][r];
    mb[64 * NO] = m;
    mb[64 * NO + 64] = l;
    __syncthreads();
    if (wv != 0) return;
#pragma unroll
    for (int w = 1; w < KW; ++w) {
      const float* ob = win_smem + w * C::MERGE + lane;
      const float m1 = ob[64 * NO], mn = fmaxf(m, m1), mu = mn == -INFINITY ? 0.f : mn;
      const float w0 = __builtin_amdgcn_exp2f(m - mu), w1 = __builtin_amdgcn_exp2f(m1 - mu);
      m = mn;
      l = l * w0 + ob[64 * NO + 64] * w1;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < NS; ++r) o[d][r] = o[d][r] * w0 + ob[64 * (NS * d + r)] * w1;
    }
  }
  float lt = l;
#pragma unroll
  for (int w = RB; w < 64; w <<= 1) lt += __shfl_xor(lt, w);
  // Row r's output, or (SPLIT) its partial slot's unnormalised dims, max and sum.
  const float inv = SPLIT ? 1.f : (lt > 0.f ? 1.f / lt : 0.f);
  auto slot = [&](int r) { return ((b * p.heads + h) * p.seq_q + r) * gridDim.y + blockIdx.y; };
  auto row_out = [&](int r) {
    return SPLIT ? p.part_acc + slot(r) * E : reinterpret_cast<float*>(p.out) + ((b * p.seq_q + r) * p.heads + h) * E;
  };
  if (SPLIT && row < L && qd == 0) {
    p.part_ml[2 * slot(row)] = m;
    p.part_ml[2 * slot(row) + 1] = lt;
  }
  bool bad = !(fabsf(lt) < INFINITY);
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < NS / 4; ++g) {
      f32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bad |= !(fabsf(o[d][4 * g + j]) < INFINITY);
        x[j] = o[d][4 * g + j] * inv;
      }
      if (row < L) *reinterpret_cast<f32x4*>(row_out(row) + RB * d + acc_row(4 * g) + 4 * qd) = x;
    }
  const uint64_t bits = __ballot(bad);
  uint32_t redo = (uint32_t)bits | (uint32_t)(bits >> 32);
  if (RB == 16) redo = (redo | redo >> 16) & 0xffffu;
  if (__builtin_expect(redo == 0, 1)) return;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  while (redo) {
    const int r = r0 + __builtin_ctz(redo);
    redo &= redo - 1;
    if (r >= L) continue;
    win_redo_row<E, uint32_t, BN>(p, wt, t0, t1, qg, kg, vg, r, [&](float rm, float rl, int d, float a) {
      row_out(r)[d] = SPLIT ? a : (rl != 0.f ? a / rl : 0.f);
      if (SPLIT && d == 0) {
        p.part_ml[2 * slot(r)] = rm;
        p.part_ml[2 * slot(r) + 1] = rl;
      }
    });
  }
}

// How a call in 32-bit MFMAs runs: key waves and rows per wave of its blocks, and splits of
// their tiles (calls of many blocks get here by their few visible keys).  128-row blocks where they give every CU one (E = 128, whose 128-key tiles leave one block
// per CU: nearly), else 32-row ones, else 16-row ones, and none of more rows than twice the
// call's (N=8 L=1 H=32 E=128 window 1023 164 -> 66).  Measured (us, window 300 unless
// noted, KW = 1 / KW = 4 RB = 32 / RB = 16): N=1 L=333 S=2500 window 512 H=12 E=64 67.5 /
// 28.1 / 20.3; N=2 L=S=700 H=12 E=64 48.0 / 24.5 / 30.7; L=S=1536 H=16 E=64 48.6 / 43.7,
// E=128 81.1 / 82.7; N=2 L=S=1024 H=16 E=128 81.8 / 102.  16-row blocks that leave half of the
// CUs idle split lists of 4 tiles or more, at least kMinShare tiles each (L=64 H=8, unsplit /
// shares of 4 / 2: E=64 window 2048 38 / 20.0 / 14.9, window 768 21.5 / 21.5 / 14.8, E=32
// window 512 10.5 / 10.5 / 10.9).
struct WinF32Plan {
  int kw, rb;
  int64_t blocks, splits;
};
constexpr int64_t kMinShare = 2;
static WinF32Plan win_f32_plan(const WindowParams& p, int E) {
  const int64_t bh = p.batch * p.heads;
  WinF32Plan w{1, 32, bh * cdiv(p.seq_q, 128), 1};
  if (w.blocks > (E == 128 ? 192 : 256) && p.seq_q > 32) return w;
  w = WinF32Plan{4, 32, bh * cdiv(p.seq_q, 32), 1};
  if (w.blocks > 256 && p.seq_q > 16) return w;
  w = WinF32Plan{4, 16, bh * cdiv(p.seq_q, 16), 1};
  const int64_t T = win_most_tiles(p, 16, 128), by_tiles = T / kMinShare;
  if (w.blocks > 0 && w.blocks <= 128 && by_tiles >= 2) w.splits = 256 / w.blocks < by_tiles ? 256 / w.blocks : by_tiles;
  w.splits = w.splits < kTiledMaxSplits ? w.splits : kTiledMaxSplits;  // what the combine merges
  return w;
}

int64_t flash_window_f32_splits(const WindowParams& p, int E) { return win_f32_plan(p, E).splits; }

template <int E, int KW, int RB, bool SPLIT>
static int win_f32_launch_t(const WindowParams& p, const WinF32Plan& w, hipStream_t stream) {
  using C = WinF32Cfg<E, KW, RB>;
  if (w.blocks > 0x7fffffff) return CA_DECLINED;
  if (C::LDS_BYTES > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(win_f32_kernel<E, KW, RB, SPLIT>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS_BYTES);
    if (e != hipSuccess) return CA_HIP_ERROR - (int)e;
  }
  hipLaunchKernelGGL((win_f32_kernel<E, KW, RB, SPLIT>), dim3((unsigned)w.blocks, (unsigned)w.splits), dim3(256),
                     C::LDS_BYTES, stream, p);
  return ca_launch_status();
}

template <int E>
static int win_f32_launch_e(const WindowParams& p, hipStream_t stream) {
  const WinF32Plan w = win_f32_plan(p, E);
  if (w.splits > 1) {
    const int st = win_f32_launch_t<E, 4, 16, true>(p, w, stream);
    return st == CA_OK ? flash_combine_launch(p, E, false, w.splits, stream) : st;
  }
  if (w.kw == 1) return win_f32_launch_t<E, 1, 32, false>(p, w, stream);
  return w.rb == 32 ? win_f32_launch_t<E, 4, 32, false>(p, w, stream) : win_f32_launch_t<E, 4, 16, false>(p, w, stream);
}

template <int E>
static int win_f32_redo(const WindowParams& p, hipStream_t stream) {
  const WinF32Plan w{1, 32, p.batch * p.heads * cdiv(p.seq_q, 128), p.redo_splits};
  if (w.splits == 1) return win_f32_launch_t<E, 1, 32, false>(p, w, stream);
  const int st = win_f32_launch_t<E, 1, 32, true>(p, w, stream);
  return st == CA_OK ? flash_combine_launch(p, E, false, w.splits, stream) : st;
}

int flash_window_f32_launch(const WindowParams& p, int E, hipStream_t stream) {
  if (!window_fits(p, E, 4)) return CA_DECLINED;
  if (p.redo) {
    switch (E) {
      case 32: return win_f32_redo<32>(p, stream);
      case 64: return win_f32_redo<64>(p, stream);
      case 128: return win_f32_redo<128>(p, stream);
    }
  }
  switch (E) {
    case 32: return win_f32_launch_e<32>(p, stream);
    case 64: return win_f32_launch_e<64>(p, stream);
    case 128: return win_f32_launch_e<128>(p, stream);
  }
  return CA_DECLINED;
}

}  // namespace ca
