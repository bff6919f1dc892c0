// The geometry of a prefill with a sliding window and sinks, and the pass that redoes single
// rows (shared by the bf16 kernel in ca_duo.h and the fp32 one in ca_win_f32.hip).
#pragma once

#include "ca_device.h"
#include "ca_internal.h"

namespace ca {

__host__ __device__ inline int imin(int a, int b) { return a < b ? a : b; }
__host__ __device__ inline int imax(int a, int b) { return a > b ? a : b; }

// The keys that a block of rows [q0, q0 + bm) walks, as a list of tiles of bn keys: tiles
// 0 .. st - 1 begin at 0, bn, ... and hold the sinks, tile i >= st begins at w0 + (i - st) bn;
// n in all.  Without a gap between sinks and window the list is one run from key 0.  The
// rows' own limits are masked in the tiles.
struct WinTiles {
  int st, w0, n;
};
__host__ __device__ inline WinTiles win_tiles(const WindowParams& p, int q0, int bm, int bn) {
  const int L = (int)p.seq_q, S = (int)p.seq_k, diag = S - L;
  const int last = (q0 + bm < L ? q0 + bm : L) - 1 + diag;  // the last row's position
  const int64_t end = (int64_t)last + p.right + 1;
  const int kend = end < 0 ? 0 : (end < S ? (int)end : S);
  const int64_t low = (int64_t)q0 + diag - p.left;
  const int klo = low < 0 ? 0 : (low < kend ? (int)low : kend);
  const int sinks = p.sinks < kend ? p.sinks : kend;
  WinTiles w{0, 0, 0};
  if (klo > sinks) {
    w.st = (sinks + bn - 1) / bn;
    w.w0 = w.st * bn > klo ? w.st * bn : klo;
  }
  w.n = w.st + (kend > w.w0 ? (kend - w.w0 + bn - 1) / bn : 0);
  return w;
}
__host__ __device__ inline int win_key0(const WinTiles& w, int tile, int bn) {
  return tile < w.st ? tile * bn : w.w0 + (tile - w.st) * bn;
}

// The split mode's share of the list (tiles [t0, t0 + share)), and the rounds that the
// wave at rows r0 .. r0 + 31 of key group grp (of kg) takes part in: nkt for the whole
// block (loads and barriers), of which it computes the nkt_w whose tiles begin before its
// last row's last key.
struct WinRounds {
  int t0, nkt, nkt_w;
};
__host__ __device__ inline WinRounds win_rounds(const WindowParams& p, const WinTiles& w, int bn, int r0, int sp, int splits,
                                                int kg, int grp) {
  const int L = (int)p.seq_q, S = (int)p.seq_k;
  const int share = (w.n + splits - 1) / splits, t0 = sp * share < w.n ? sp * share : w.n;
  const int t1 = t0 + share < w.n ? t0 + share : w.n;
  const int64_t end = (int64_t)r0 + 32 + S - L + p.right;
  const int kend = r0 >= L || end < 0 ? 0 : (end < S ? (int)end : S);
  const int head = (kend + bn - 1) / bn;  // sink tiles that begin before kend, if no window tile does
  const int before = kend > w.w0 ? w.st + (kend - w.w0 + bn - 1) / bn : (head < w.st ? head : w.st);
  const int tw = before < t1 ? before : t1;
  WinRounds r;
  r.t0 = t0;
  r.nkt = (t1 - t0 + kg - 1) / kg;
  r.nkt_w = tw - t0 - grp > 0 ? (tw - t0 - grp + kg - 1) / kg : 0;
  return r;
}

// What the kernels take: 32-bit positions, and (bf16) a tile's 64 rows within 32-bit byte
// offsets; larger strides are declined and the caller copies the tensor.
inline bool window_fits(const WindowParams& p, int E, int esize) {
  int64_t ts = p.ks[1] > p.vs[1] ? p.ks[1] : p.vs[1];
  if (p.qs[1] > ts) ts = p.qs[1];
  return p.qs[1] >= 0 && p.ks[1] >= 0 && p.vs[1] >= 0 && 64 * (ts + E) * esize < ((int64_t)1 << 31) &&
         p.seq_q <= kWindowMaxSeq && p.seq_k <= kWindowMaxSeq;
}

// The most tiles of any block: what the plans go by.
__host__ __device__ inline int64_t win_most_tiles(const WindowParams& p, int bm, int bn) {
  const int64_t seen = (int64_t)p.left + p.right + bm;
  const int64_t all = cdiv(p.seq_k, bn), some = cdiv(seen, bn) + cdiv(p.sinks < p.seq_k ? p.sinks : p.seq_k, bn);
  return all < some ? all : some;
}

// Whether the first blocks have less to do than the last ones, as in a causal call of fewer
// than twice as many keys as rows, over a window of `tenths` tenths of the keys or more:
// pairs of blocks do even it out then.
inline bool win_triangle(const WindowParams& p, int tenths) {
  return p.right < p.seq_q - 1 && p.seq_k < 2 * p.seq_q && 10 * ((int64_t)p.left + 1) >= tenths * p.seq_k;
}

// Whether the row at position pos sees key j (of 0 .. S - 1).
__host__ __device__ inline bool win_sees(const WindowParams& p, int pos, int j) {
  return j <= (int64_t)pos + p.right && (j >= (int64_t)pos - p.left || j < p.sinks);
}

// Row `row` of (b, h) by one wave, key by key: what the matrix kernels leave to redo.  They
// weigh a key that a row does not see with 0, and 0 times an infinity or a NaN in its V is
// NaN; here such keys are not touched.  Rows that come out not finite are rare, or the
// inputs are wrong: a lane takes a key of each tile for the logit and E / 64 dims (lanes
// below 32 for E = 32) for the sum, and a row whose every dim is NaN ends there (inputs of
// NaNs would otherwise take this path over all of their keys).  T: 16-bit (bf16) or 32-bit
// (fp32) words.  Tiles [t0, t1) of the list, of BN keys; the scaled log2 max m, sum l and
// the unnormalised dims go to `store(m, l, dim, acc)`.
template <int E, typename T, int BN, typename F>
__device__ __forceinline__ void win_redo_row(const WindowParams& p, const WinTiles& w, int t0, int t1, const T* q,
                                             const T* k, const T* v, int row, F&& store) {
  constexpr int DPC = E >= 64 ? E / 64 : 1, PER = 16 / sizeof(T), AHEAD = 8;
  auto f32 = [](T x) { return __uint_as_float(sizeof(T) == 2 ? (uint32_t)x << 16 : (uint32_t)x); };
  const int lane = threadIdx.x & 63, S = (int)p.seq_k, pos = row + S - (int)p.seq_q;
  const bool dims = lane * DPC < E;
  const T* qr = q + row * p.qs[1];
  float m = -INFINITY, l = 0.f, acc[DPC];
#pragma unroll
  for (int i = 0; i < DPC; ++i) acc[i] = 0.f;
#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
#pragma unroll 1
    for (int c0 = 0; c0 < BN; c0 += kWave) {
      const int k0 = win_key0(w, t, BN) + c0, j = k0 + lane;
      const bool seen = c0 + lane < BN && j < S && win_sees(p, pos, j);
      float x = -INFINITY;
      if (seen) {
        x = 0.f;
#pragma unroll 4
        for (int d = 0; d < E; d += PER) {  // 16 bytes of K and of q
          const u32x4 kq = *reinterpret_cast<const u32x4*>(k + j * p.ks[1] + d);
          const u32x4 qq = *reinterpret_cast<const u32x4*>(qr + d);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a = kq[i], b = qq[i];
            if (sizeof(T) == 2) {
              x = fmaf(bf16_lo(a), bf16_lo(b), x);
              x = fmaf(bf16_hi(a), bf16_hi(b), x);
            } else {
              x = fmaf(__uint_as_float(a), __uint_as_float(b), x);
            }
          }
        }
        x *= p.c;
        x = x != x ? INFINITY : x;  // a NaN logit: NaN below (inf - inf)
      }
      const float mn = fmaxf(m, wave_max(x)), mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - mu), e = seen ? __builtin_amdgcn_exp2f(x - mu) : 0.f;
      m = mn;
      l = l * alpha + wave_sum(e);
#pragma unroll
      for (int i = 0; i < DPC; ++i) acc[i] *= alpha;
      uint64_t todo = __ballot(seen);
#pragma unroll 1
      while (todo) {  // AHEAD visible keys at a time, their V rows loaded before any is used
        float pu[AHEAD], vu[AHEAD][DPC];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          const int u = todo ? __builtin_ctzll(todo) : -1;
          todo &= todo - 1;
          pu[a] = u < 0 ? 0.f : __shfl(e, u);
#pragma unroll
          for (int i = 0; i < DPC; ++i)
            vu[a][i] = u >= 0 && dims ? f32(v[(k0 + u) * p.vs[1] + lane * DPC + i]) : 0.f;
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
#pragma unroll
          for (int i = 0; i < DPC; ++i) acc[i] = fmaf(pu[a], vu[a][i], acc[i]);
      }
    }
    bool lost = true;
#pragma unroll
    for (int i = 0; i < DPC; ++i) lost &= acc[i] != acc[i];
    if (!__any(dims && !lost)) break;
  }
  if (dims) {
#pragma unroll
    for (int i = 0; i < DPC; ++i) store(m, l, lane * DPC + i, acc[i]);
  }
}

}  // namespace ca
