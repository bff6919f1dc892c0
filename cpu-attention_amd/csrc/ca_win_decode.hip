// Paged decode of one query token per sequence with a sliding window and sinks, over
// the package's bf16 / fp32 cache or over its 8-bit one.
//
// The newest of len tokens sees keys [lo, len), lo = max(0, len - 1 - left) (left < 0:
// lo = 0), and the sinks [0, min(sinks, lo)).  Logits, the base-2 online softmax, fp32
// accumulation and the output are ca_decode.hip's.  An 8-bit cache holds e4m3 codes, one
// power-of-two scale per (page, head) for K and one for V: K's scale goes into the
// logits' factor, V's into the probability that weighs the row, so a code costs its
// conversion alone.
//
// Only what the row sees is walked: the 16-key units that hold a sink or a window key,
// numbered without the gap between them (Span).  The grid covers the most units that a
// row of the call's window can have, not the page table's capacity.  One wave takes a
// tile of TK keys (TK / 16 units), a block 8 tiles; a unit's visible keys are 16 bits of
// a mask, which decides what is read: a masked key's V row is never loaded, and its
// logit is -inf whatever its K holds.
//
// Bound: reading the visible keys once (HBM).
#include "ca_device.h"
#include "ca_internal.h"
#include "ca_merge.h"

namespace ca {

constexpr int kUnit = 16;     // keys per unit: never straddles a page
constexpr int kWinTile = 64;  // keys per tile

// The units that row `seq` walks: units 0 .. su - 1 hold the sinks, unit i >= su of the
// walk is unit i - su + u0 of the sequence; nu in all.
struct Span {
  int64_t len, lo, s, su, u0, nu;
};
__device__ __forceinline__ Span span_of(const WinDecodeParams& p, int64_t seq) {
  const int64_t cap = p.pt_width * p.page;
  Span x;
  x.len = (int64_t)p.lens[seq] + p.len_add;
  x.len = x.len < 0 ? 0 : (x.len < cap ? x.len : cap);
  x.lo = p.left < 0 ? 0 : max<int64_t>(0, x.len - 1 - p.left);
  x.s = min<int64_t>(p.sinks, x.lo);
  x.su = cdiv(x.s, kUnit);
  x.u0 = max<int64_t>(x.lo / kUnit, x.su);
  x.nu = x.su + max<int64_t>(0, cdiv(x.len, kUnit) - x.u0);
  return x;
}

// The low n bits (n <= 0: none, n >= 16: all of a unit).
__device__ __forceinline__ uint32_t low_bits(int64_t n) {
  return n <= 0 ? 0u : (n >= kUnit ? 0xffffu : (1u << (int)n) - 1u);
}

template <int E, bool BF, bool F8>
struct WinShape {
  static constexpr int CES = F8 ? 1 : (BF ? 2 : 4);  // bytes of a cache element
  static constexpr int W = E * CES / 4;              // K words per key
  static constexpr int DPL = 16 / CES;               // V elements per 16-byte load
  static constexpr int LPR = E / DPL;                // lanes per V row
  static constexpr int G = kWave / LPR;              // V rows per wave load
};

// Tile `tile` (units tile * TK / 16 ...) of row (seq, h): leaves the wave's partial
// state (P.V, max in scaled log2 units, sum) in part[E + 2].
template <int E, bool BF, bool F8, int TK>
__device__ __forceinline__ void win_tile(const WinDecodeParams& p, const Span& sp, int64_t seq, int64_t h, int64_t tile,
                                         float* p_lds, float* part) {
  using D = WinShape<E, BF, F8>;
  constexpr int W = D::W, DPL = D::DPL, LPR = D::LPR, G = D::G, CES = D::CES;
  constexpr int NU = TK / kUnit, NQ = TK / 4, SPLIT = kWave / NQ, WPL = W / SPLIT;
  static_assert(TK == 64, "one 64-bit mask of visible keys");
  const int lane = threadIdx.x & 63;
  const int quad = lane % NQ, phase = lane / NQ;  // key quad of the tile, words phase, phase + SPLIT, ...

  // Lane u < NU: unit u's visible keys, its page's first K word and V element, its scales.
  int64_t kb = 0, vb = 0;
  uint32_t vis = 0;
  float ksc = 1.f, vsc = 1.f;
  const int64_t iu = tile * NU + lane;
  if (lane < NU && iu < sp.nu) {
    const int64_t tu = (iu < sp.su ? iu : iu - sp.su + sp.u0) * kUnit;
    const int64_t pi = tu / p.page, off = tu - pi * p.page;
    const int64_t blk = p.page_table[seq * p.pt_width + pi];
    if (blk >= 0 && blk < p.nblocks) {
      vis = low_bits(sp.len - tu) & (low_bits(sp.s - tu) | ~low_bits(sp.lo - tu));
      const int64_t bh = blk * p.heads + h, base = bh * p.page;
      kb = base * W + off;
      vb = (base + off) * E;
      if (F8) {
        ksc = p.k_scale[bh];
        vsc = p.v_scale[bh];
      }
    }
  }
  uint64_t mask = 0;
#pragma unroll
  for (int u = 0; u < NU; ++u) mask |= (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)vis, u) << (kUnit * u);

  // ---- Q.K
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  const uint32_t qvis = (uint32_t)(mask >> (4 * quad)) & 15u;
  const int64_t kbu = __shfl(kb, quad >> 2);
  float cs = p.c;
  if (F8) cs *= __shfl(ksc, quad >> 2);
  if (qvis) {
    const uint32_t* kp = p.kc + kbu + 4 * (quad & 3) + (int64_t)phase * p.page;
    constexpr int QU = WPL < 16 ? WPL : 16;  // K loads in flight
    for (int w0 = 0; w0 < WPL; w0 += QU) {
      u32x4 k4[QU];
#pragma unroll
      for (int i = 0; i < QU; ++i)
        k4[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + (int64_t)(w0 + i) * SPLIT * p.page));
#pragma unroll
      for (int i = 0; i < QU; ++i) {
        const int w = phase + (w0 + i) * SPLIT;
        if constexpr (F8) {
          float q4[4];
          if constexpr (BF) {
            const u32x2 qw = *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint16_t*>(p.q) + seq * p.q_stride +
                                                             h * E + 4 * w);
            q4[0] = bf16_lo(qw.x);
            q4[1] = bf16_hi(qw.x);
            q4[2] = bf16_lo(qw.y);
            q4[3] = bf16_hi(qw.y);
          } else {
            const f32x4 qw = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p.q) + seq * p.q_stride +
                                                             h * E + 4 * w);
#pragma unroll
            for (int x = 0; x < 4; ++x) q4[x] = qw[x];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t kw = k4[i][j];
            const f32x2 lo = e4m3_lo(kw), hi = e4m3_hi(kw);
            s[j] = fmaf(lo.x, q4[0], s[j]);
            s[j] = fmaf(lo.y, q4[1], s[j]);
            s[j] = fmaf(hi.x, q4[2], s[j]);
            s[j] = fmaf(hi.y, q4[3], s[j]);
          }
        } else if constexpr (BF) {
          const uint32_t qw = (reinterpret_cast<const uint32_t*>(p.q) + (seq * p.q_stride + h * E) / 2)[w];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t kw = k4[i][j];
            s[j] = __builtin_amdgcn_fdot2_f32_bf16(as_bf16x2(kw), as_bf16x2(qw), s[j], false);
          }
        } else {
          const float qw = (reinterpret_cast<const float*>(p.q) + seq * p.q_stride + h * E)[w];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t kw = k4[i][j];
            s[j] = fmaf(__uint_as_float(kw), qw, s[j]);
          }
        }
      }
    }
  }
  // The SPLIT lanes of a quad sum their parts.  Scaled logits: -inf for a masked key,
  // +inf for a NaN (its row comes out NaN then; as a NaN, the maxima would skip it and
  // a tile of nothing else would count as empty).
  float x[4], mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int o = NQ; o < kWave; o <<= 1) s[j] += __shfl_xor(s[j], o);
    x[j] = s[j] * cs;
    x[j] = x[j] != x[j] ? INFINITY : x[j];
    x[j] = qvis >> j & 1 ? x[j] : -INFINITY;
    mx = fmaxf(mx, x[j]);
  }
  const float m = wave_max(mx), mu = m == -INFINITY ? 0.f : m;
  float pr[4], ls = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    pr[j] = __builtin_amdgcn_exp2f(x[j] - mu);
    ls += pr[j];
  }
  const float l = wave_sum(phase == 0 ? ls : 0.f);  // one lane per quad counts it
  if (F8) {
    const float vq = __shfl(vsc, quad >> 2);
#pragma unroll
    for (int j = 0; j < 4; ++j) pr[j] *= vq;
  }
  wave_lds_sync();
  if (phase == 0) *reinterpret_cast<f32x4*>(&p_lds[4 * quad]) = f32x4{pr[0], pr[1], pr[2], pr[3]};
  wave_lds_sync();

  // ---- P.V: lane group g reads rows g, g + G, ... of the tile, lane dl of it 16 bytes.
  constexpr int R = TK / G, B = R < 16 ? R : 16;
  const int g = lane / LPR, dl = lane - g * LPR;
  const char* vbase = reinterpret_cast<const char*>(p.vc) + dl * 16;
  float acc[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = 0.f;
#pragma unroll
  for (int b0 = 0; b0 < R; b0 += B) {
    u32x4 v4[B];
    bool ok[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int key = g + G * (b0 + i);
      ok[i] = mask >> key & 1;
      const int64_t vu = __shfl(vb, key / kUnit);
      if (ok[i])
        v4[i] = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4*>(vbase + (vu + (int64_t)(key & (kUnit - 1)) * E) * CES));
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (ok[i]) {
        const float pj = p_lds[g + G * (b0 + i)];
#pragma unroll
        for (int x4 = 0; x4 < 4; ++x4) {
          const uint32_t vw = v4[i][x4];
          if constexpr (F8) {
            const f32x2 lo = e4m3_lo(vw), hi = e4m3_hi(vw);
            acc[4 * x4] = fmaf(pj, lo.x, acc[4 * x4]);
            acc[4 * x4 + 1] = fmaf(pj, lo.y, acc[4 * x4 + 1]);
            acc[4 * x4 + 2] = fmaf(pj, hi.x, acc[4 * x4 + 2]);
            acc[4 * x4 + 3] = fmaf(pj, hi.y, acc[4 * x4 + 3]);
          } else if constexpr (BF) {
            acc[2 * x4] = fmaf(pj, bf16_lo(vw), acc[2 * x4]);
            acc[2 * x4 + 1] = fmaf(pj, bf16_hi(vw), acc[2 * x4 + 1]);
          } else {
            acc[x4] = fmaf(pj, __uint_as_float(vw), acc[x4]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = LPR; o < kWave; o <<= 1)
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[i] += __shfl_xor(acc[i], o);
  if (lane < LPR) {
#pragma unroll
    for (int i = 0; i < DPL; ++i) part[lane * DPL + i] = acc[i];
  }
  if (lane == 0) {
    part[E] = m;
    part[E + 1] = l;
  }
}

template <int E, bool BF, bool F8, int TK>
__global__ __launch_bounds__(64 * kDecWaves) void win_decode_kernel(WinDecodeParams p) {
  __shared__ __attribute__((aligned(16))) float p_lds[kDecWaves][TK];
  __shared__ float part[kDecWaves][E + 2];
  constexpr int NU = TK / kUnit;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  const int64_t s = row / p.heads, h = row - s * p.heads;
  const int64_t tile = (int64_t)blockIdx.y * kDecWaves + wv;
  const Span sp = span_of(p, s);
  // Waves past the row's last unit exit (the barrier below waits for the others only);
  // the row's first wave stays, and writes a row with no key as exactly 0.
  if (tile * NU >= sp.nu && tile != 0) return;
  win_tile<E, BF, F8, TK>(p, sp, s, h, tile, p_lds[wv], part[wv]);
  __syncthreads();
  if (wv != 0) return;
  constexpr int DPC = E >= 64 ? E / 64 : 1;
  const int lane = threadIdx.x & 63;
  const int64_t tiles = max<int64_t>(1, cdiv(sp.nu, NU));
  const int n = (int)min<int64_t>(kDecWaves, tiles - (int64_t)blockIdx.y * kDecWaves);
  float mx, acc[DPC];
  const float l = merge_states<E, DPC>(n, [&](int t, int i) {
    return part[t][i == -1 ? E : (i == -2 ? E + 1 : i)];
  }, mx, acc);
  if (tiles <= kDecWaves) {
    if (lane * DPC < E) store_out<DPC, BF>(p.out, row * E + lane * DPC, acc, l > 0.f ? 1.f / l : 0.f);
    return;
  }
  const int64_t slot = row * cdiv(p.tiles, kDecWaves) + blockIdx.y;
  if (lane * DPC < E) {
#pragma unroll
    for (int i = 0; i < DPC; ++i) p.part_acc[slot * E + lane * DPC + i] = acc[i];
  }
  if (lane == 0) {
    p.part_ml[2 * slot] = mx;
    p.part_ml[2 * slot + 1] = l;
  }
}

// One wave per row of more than one block: merges the blocks' partials.
template <int E, bool BF, int TK>
__global__ __launch_bounds__(256) void win_decode_combine_kernel(WinDecodeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= p.nseqs * p.heads) return;
  const int64_t tiles = cdiv(span_of(p, row / p.heads).nu, TK / kUnit);
  if (tiles <= kDecWaves) return;  // written by its block
  merge_partials<E, BF, false>(p, row, (int)cdiv(tiles, kDecWaves), lane);
}

// The most tiles that a row can have: its page table's capacity, or the units of the
// sinks and of a window that begins at any key of its first unit.
int64_t win_decode_tiles(int64_t pt_width, int64_t page, int64_t left, int64_t sinks) {
  int64_t units = pt_width * page / kUnit;
  if (left >= 0) {
    const int64_t seen = cdiv(sinks, kUnit) + cdiv(left + kUnit, kUnit);
    units = units < seen ? units : seen;
  }
  return cdiv(units, kWinTile / kUnit);
}

// Partial slots: one per (row, block of 8 tiles) when rows can outgrow one block.
int64_t win_decode_slots(int64_t rows, int64_t tiles) { return tiles > kDecWaves ? rows * cdiv(tiles, kDecWaves) : 0; }

template <int E, bool BF, bool F8>
static int win_decode_launch_t(const WinDecodeParams& p, hipStream_t stream) {
  const int64_t rows = p.nseqs * p.heads;
  const int64_t gy = p.tiles > kDecWaves ? cdiv(p.tiles, kDecWaves) : 1;
  if (rows > 0x7fffffff || gy > 65535 || win_decode_slots(rows, p.tiles) > p.slots) return CA_DECLINED;
  hipLaunchKernelGGL((win_decode_kernel<E, BF, F8, kWinTile>), dim3((unsigned)rows, (unsigned)gy), dim3(64 * kDecWaves),
                     0, stream, p);
  const int st = ca_launch_status();
  if (st != CA_OK || gy == 1) return st;
  hipLaunchKernelGGL((win_decode_combine_kernel<E, BF, kWinTile>), dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, stream, p);
  return ca_launch_status();
}

template <bool BF, bool F8>
static int win_decode_launch_e(const WinDecodeParams& p, int E, hipStream_t stream) {
  switch (E) {
    case 32: return win_decode_launch_t<32, BF, F8>(p, stream);
    case 64: return win_decode_launch_t<64, BF, F8>(p, stream);
    case 128: return win_decode_launch_t<128, BF, F8>(p, stream);
  }
  return CA_DECLINED;
}

int win_decode_launch(const WinDecodeParams& p, int E, int bf16, hipStream_t stream) {
  if (p.nseqs == 0) return CA_OK;
  if (p.k_scale)
    return bf16 ? win_decode_launch_e<true, true>(p, E, stream) : win_decode_launch_e<false, true>(p, E, stream);
  return bf16 ? win_decode_launch_e<true, false>(p, E, stream) : win_decode_launch_e<false, false>(p, E, stream);
}

}  // namespace ca
