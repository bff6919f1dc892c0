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
// tile of TK keys (TK / 16 units), a block 8 tiles, merged in LDS; a row of more blocks is
// merged by its last one, or (many rows or blocks) by a second kernel.  A unit's visible
// keys are 16 bits of a mask, which decides what is read: a masked key's V row is never
// loaded, and its logit is -inf whatever its K holds.
//
// Bound: reading the visible keys once (HBM).
#include "ca_device.h"
#include "ca_fp8.h"
#include "ca_internal.h"
#include "ca_merge.h"

namespace ca {

constexpr int kUnit = 16;     // keys per unit: never straddles a page
constexpr int kWinTile = 64;  // keys per tile
// V rows of a lane up to which they are loaded before the logits: 2 (8-bit E = 32) hide a
// load's latency for few registers.  4 take 8-bit E = 64 from 64 to 99 registers, two blocks
// per CU instead of three (N=64 H=32, lengths to 4095: 107 -> 136 us), 8 leave 8-bit E = 128
// one (193 -> 284 us).
constexpr int kEarlyRows = 2;

// Positions and pages fit 32 unsigned bits (lengths are 32-bit, plus at most 2^30 new
// tokens; the launcher bounds the page), and a 32-bit division takes a third of a 64-bit one.
__device__ __forceinline__ int64_t page_of(int64_t pos, int64_t page) { return (uint32_t)pos / (uint32_t)page; }

// The units that row `seq` walks: units 0 .. su - 1 hold the sinks, unit i >= su of the
// walk is unit i - su + u0 of the sequence; nu in all.
//
// The walk's tiles take TK / 16 units each, the last one the units from `last` on.  A call
// that appends to an 8-bit cache in this kernel (FOLD) gives the last page's units, at
// most 4, a tile of their own: the wave that takes it may rescale the page, and nobody else
// may read it then.
struct Span {
  int64_t len, lo, s, su, u0, nu, last, tiles;
};
template <bool FOLD>
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
  constexpr int NU = kWinTile / kUnit;
  if (FOLD) {
    const int64_t lp = x.len > 0 ? page_of(x.len - 1, p.page) * (p.page / kUnit) : 0;  // the last page's first unit
    x.last = lp < x.su ? lp : x.su + max<int64_t>(0, lp - x.u0);
    x.tiles = cdiv(x.last, NU) + 1;
  } else {
    x.last = x.nu > 0 ? (x.nu - 1) / NU * NU : 0;
    x.tiles = x.last / NU + 1;
  }
  return x;
}

// The largest length, 0 if that is negative.
__device__ __forceinline__ int64_t longest_of(const WinDecodeParams& p) {
  int32_t longest = 0;
  for (int64_t i = threadIdx.x & 63; i < p.nseqs; i += kWave) longest = max(longest, p.lens[i]);
#pragma unroll
  for (int d = kWave / 2; d; d /= 2) longest = max(longest, __shfl_xor(longest, d));
  return longest;
}

// The low n bits (n <= 0: none, n >= 16: all of a unit).
__device__ __forceinline__ uint32_t low_bits(int64_t n) {
  return n <= 0 ? 0u : (n >= kUnit ? 0xffffu : (1u << (int)n) - 1u);
}

// The sums of v[0 .. N) over the lanes that differ in the bits FIRST, 2 FIRST, .. 32 of their
// number.  At each bit a lane passes half of its values on and adds the other half of its
// neighbour's (N - 1 exchanges instead of N times the bits): it ends with the sums of
// v[at ..), max(1, N FIRST / 64) of them in v[0 ..), and returns at.
template <int N, int FIRST, int A>
__device__ __forceinline__ int fold_lanes(float (&v)[A], int lane) {
  if constexpr (FIRST >= kWave) {
    return 0;
  } else if constexpr (N > 1) {
    constexpr int H = N / 2;
    const bool up = lane & FIRST;
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float lo = v[i], hi = v[H + i];
      v[i] = (up ? hi : lo) + __shfl_xor(up ? lo : hi, FIRST);
    }
    return (up ? H : 0) + fold_lanes<H, 2 * FIRST>(v, lane);
  } else {
    v[0] += __shfl_xor(v[0], FIRST);
    return fold_lanes<1, 2 * FIRST>(v, lane);
  }
}

template <int E, bool BF, bool F8>
struct WinShape {
  static constexpr int CES = F8 ? 1 : (BF ? 2 : 4);  // bytes of a cache element
  static constexpr int W = E * CES / 4;              // K words per key
  static constexpr int DPL = 16 / CES;               // V elements per 16-byte load
  static constexpr int LPR = E / DPL;                // lanes per V row
  static constexpr int G = kWave / LPR;              // V rows per wave load
};

// Tile `tile` of row (seq, h): leaves the wave's partial state (P.V, max in scaled log2
// units, sum) in part[E + 2].  APPEND: the row's last tile stores the call's new token.
template <int E, bool BF, bool F8, bool APPEND, int TK>
__device__ __forceinline__ void win_tile(const WinDecodeParams& p, const Span& sp, int64_t seq, int64_t h, int64_t tile,
                                         float* p_lds, float* part, uint32_t* kl) {
  using D = WinShape<E, BF, F8>;
  constexpr int W = D::W, DPL = D::DPL, LPR = D::LPR, G = D::G, CES = D::CES;
  constexpr int NU = TK / kUnit, NQ = TK / 4, SPLIT = kWave / NQ, WPL = W / SPLIT;
  static_assert((TK == 64 || TK == 128) && W % SPLIT == 0, "tile shape");
  const int lane = threadIdx.x & 63;
  const int quad = lane % NQ, phase = lane / NQ;  // key quad of the tile, words phase, phase + SPLIT, ...

  // Lane u < NU: unit u's visible keys, its page's first K word and V element, its scales.
  int64_t kb = 0, vb = 0;
  uint32_t vis = 0;
  float ksc = 1.f, vsc = 1.f;
  const bool final = tile == sp.tiles - 1;
  const int64_t iu = (final ? sp.last : tile * NU) + lane;
  // The new token: at position lens[seq], the row's newest unless that lies past the table.
  // A host that has such lengths refused (longest) wants no sequence's token stored then.
  bool fresh = APPEND && final && sp.len > 0 && p.lens[seq] == sp.len - 1;
  if (APPEND && fresh && p.longest && p.nseqs > 1) fresh = longest_of(p) < p.pt_width * p.page;
  if constexpr (APPEND && F8) {
    if (fresh) {
      const int64_t pi = page_of(sp.len - 1, p.page), at = sp.len - 1 - pi * p.page;
      const int64_t blk = p.page_table[seq * p.pt_width + pi];
      if (blk >= 0 && blk < p.nblocks) {
        Store8Page s;
        s.key = p.k_new;
        s.value = p.v_new;
        s.tok_stride = p.new_stride;
        s.kc = p.kc_store;
        s.vc = p.vc_store;
        s.k_scale = p.k_scale_store;
        s.v_scale = p.v_scale_store;
        s.heads = p.heads;
        s.page = p.page;
        store_page<E, BF>(s, blk, h, kl, [&](int64_t t) -> int { return t == at ? (int)seq : -1; });
        // The codes and scales are read back below, by other lanes.
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
      }
    }
  }
  if (lane < NU && iu < sp.nu && (final || lane < sp.last - tile * NU)) {
    const int64_t tu = (iu < sp.su ? iu : iu - sp.su + sp.u0) * kUnit;
    const int64_t pi = page_of(tu, p.page), off = tu - pi * p.page;
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
  uint64_t mask[TK / 64] = {};  // the tile's visible keys
#pragma unroll
  for (int u = 0; u < NU; ++u)
    mask[u / 4] |= (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)vis, u) << (kUnit * (u % 4));

  // The new token of a 16- or 32-bit cache: its words and q's, and its key in the tile.  Its
  // logit comes from these registers and its V row from where it lies, so nothing waits
  // for the stores to the cache.
  constexpr int KNW = (W + kWave - 1) / kWave;
  uint32_t knw[KNW], qnw[KNW];
  const char* vnew = nullptr;
  int newj = -1;
  if constexpr (APPEND && !F8) {
    const int last = (int)(sp.nu - 1 - sp.last);  // the tile's last unit holds it
    if (fresh && __builtin_amdgcn_readlane((int)vis, last & (NU - 1)) != 0) {
      newj = kUnit * last + (int)((sp.len - 1) & (kUnit - 1));
      const int64_t src = seq * p.new_stride + h * E;
      const uint32_t* kn = reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(p.k_new) + src * CES);
      const uint32_t* qw = reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(p.q) + (seq * p.q_stride + h * E) * CES);
      vnew = reinterpret_cast<const char*>(p.v_new) + src * CES;
      const int64_t kbn = __shfl(kb, last), vbn = __shfl(vb, last);
      const int x = newj & (kUnit - 1);
#pragma unroll
      for (int i = 0; i < KNW; ++i) {
        const int w = lane + kWave * i;
        knw[i] = w < W ? kn[w] : 0u;
        qnw[i] = w < W ? qw[w] : 0u;
        if (w < W) p.kc_store[kbn + (int64_t)w * p.page + x] = knw[i];
      }
      if (lane < W / 4)
        *reinterpret_cast<u32x4*>(p.vc_store + (vbn + (int64_t)x * E) * CES / 4 + 4 * lane) =
            *reinterpret_cast<const u32x4*>(vnew + 16 * lane);
    }
  }

  // V rows: lane group g reads rows g, g + G, ... of the tile, lane dl of it 16 bytes.  Where
  // a lane's rows fit the registers (EARLY) they are loaded before the logits, beside K.
  constexpr int R = TK / G, B = R < 16 ? R : 16;
  constexpr bool EARLY = R <= kEarlyRows;
  const int g = lane / LPR, dl = lane - g * LPR;
  u32x4 v4[B];
  auto load_v = [&](int b0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int key = g + G * (b0 + i);
      const int64_t vu = __shfl(vb, key / kUnit);
      const char* at = reinterpret_cast<const char*>(p.vc) + (vu + (int64_t)(key & (kUnit - 1)) * E) * CES;
      if (APPEND && !F8 && key == newj) at = vnew;
      if (mask[G * (b0 + i) / 64] >> (key % 64) & 1) v4[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at + dl * 16));
    }
  };

  // ---- Q.K
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  const uint32_t qvis = (uint32_t)(mask[TK == 64 || quad < 16 ? 0 : 1] >> (4 * (quad % 16))) & 15u;
  const int64_t kbu = __shfl(kb, quad >> 2);
  float cs = p.c;
  if (F8) cs *= __shfl(ksc, quad >> 2);
  constexpr int QU = WPL < 16 ? WPL : 16;  // K loads in flight
  u32x4 k4[QU];
  const uint32_t* kp = p.kc + kbu + 4 * (quad & 3) + (int64_t)phase * p.page;
  auto load_k = [&](int w0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QU; ++i)
      k4[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + (int64_t)(w0 + i) * SPLIT * p.page));
  };
  if (qvis) load_k(0);
  if (EARLY) load_v(0);
  if (qvis) {
    for (int w0 = 0; w0 < WPL; w0 += QU) {
      if (w0 > 0) load_k(w0);
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
  float lnew = 0.f;
  if constexpr (APPEND && !F8) {
    if (newj >= 0) {
#pragma unroll
      for (int i = 0; i < KNW; ++i) {
        if constexpr (BF)
          lnew = __builtin_amdgcn_fdot2_f32_bf16(as_bf16x2(knw[i]), as_bf16x2(qnw[i]), lnew, false);
        else
          lnew = fmaf(__uint_as_float(knw[i]), __uint_as_float(qnw[i]), lnew);
      }
      lnew = wave_sum(lnew);
    }
  }
  // The SPLIT lanes of a quad sum their parts, each ending with the logits of KPL of its keys,
  // 4 quad + j0 ...  Scaled logits: -inf for a masked key, +inf for a NaN (its row comes out
  // NaN then; as a NaN, the maxima would skip it and a tile of nothing else would count as
  // empty).
  constexpr int KPL = 4 / SPLIT;
  const int j0 = fold_lanes<4, NQ>(s, lane);
  float x[KPL], mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < KPL; ++j) {
    if (APPEND && !F8 && 4 * quad + j0 + j == newj) s[j] = lnew;
    x[j] = s[j] * cs;
    x[j] = x[j] != x[j] ? INFINITY : x[j];
    x[j] = qvis >> (j0 + j) & 1 ? x[j] : -INFINITY;
    mx = fmaxf(mx, x[j]);
  }
  const float m = wave_max(mx), mu = m == -INFINITY ? 0.f : m;
  float pr[KPL], ls = 0.f;
#pragma unroll
  for (int j = 0; j < KPL; ++j) {
    pr[j] = __builtin_amdgcn_exp2f(x[j] - mu);
    ls += pr[j];
  }
  const float l = wave_sum(ls);
  if (F8) {
    const float vq = __shfl(vsc, quad >> 2);
#pragma unroll
    for (int j = 0; j < KPL; ++j) pr[j] *= vq;
  }
#pragma unroll
  for (int j = 0; j < KPL; ++j) p_lds[4 * quad + j0 + j] = pr[j];
  wave_lds_sync();

  // ---- P.V
  float acc[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = 0.f;
#pragma unroll
  for (int b0 = 0; b0 < R; b0 += B) {
    if (!EARLY) load_v(b0);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (mask[G * (b0 + i) / 64] >> ((g + G * (b0 + i)) % 64) & 1) {
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
  // The lane groups sum theirs: a lane ends with NP dims of its 16 bytes (the same ones as
  // another lane's, where the groups outnumber the dims).
  constexpr int NP = DPL > G ? DPL / G : 1;
  const int d0 = dl * DPL + fold_lanes<DPL, LPR>(acc, lane);
#pragma unroll
  for (int i = 0; i < NP; ++i) part[d0 + i] = acc[i];
  if (lane == 0) {
    part[E] = m;
    part[E + 1] = l;
  }
}

// In-kernel merge of a row's nrow blocks: this block's partial (mx, l, acc) goes to `slot`
// and the row's last block writes the row.
//
// The row's counter word holds the call's tag (high 32 bits) and the blocks counted so far
// (low 32).  A word with another tag (a fresh workspace's contents, or 0, which the last
// block leaves behind and no call's tag is) is first made the tag with none counted:
// `seen` is the word as this block read it, and where that swap fails another block's has
// succeeded.  Then every block adds itself once, so nothing is tried again however many
// finish together.
//
// The partial is written with agent-scope atomic stores, which the hardware makes visible
// device-wide (they write through the XCD's L2) by the time the wave's store counter
// reaches zero; only then does the block count itself in.  The block that completes the
// count has seen every other block's count, hence every other partial, and reads them with
// agent-scope atomic loads: no L2 write-back or invalidation, which agent-scope fences
// would do for the whole L2.
template <int E, bool BF, int DPC>
__device__ __forceinline__ void merge_in_last_block(const DecodeParams& p, int64_t row, int64_t slot, int nrow, uint64_t seen,
                                                    float mx, float l, const float (&acc)[DPC], int lane) {
  uint64_t* ctr = p.counters + row;
  if (lane == 0 && (uint32_t)(seen >> 32) != p.tag)
    __hip_atomic_compare_exchange_strong(ctr, &seen, (uint64_t)p.tag << 32, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
  if (lane * DPC < E) {
#pragma unroll
    for (int i = 0; i < DPC; ++i)
      __hip_atomic_store(p.part_acc + slot * E + lane * DPC + i, acc[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (lane == 0) {
    __hip_atomic_store(p.part_ml + 2 * slot, mx, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(p.part_ml + 2 * slot + 1, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  int arrived = 0;
  if (lane == 0) arrived = (int)(uint32_t)__hip_atomic_fetch_add(ctr, (uint64_t)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
  arrived = __builtin_amdgcn_readfirstlane(arrived);
  if (arrived != nrow) return;
  asm volatile("" ::: "memory");
  if (lane == 0) __hip_atomic_store(ctr, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  merge_partials<E, BF, true>(p, row, nrow, lane);
}

template <int E, bool BF, bool F8, bool APPEND, int TK>
__global__ __launch_bounds__(64 * kDecWaves) void win_decode_kernel(WinDecodeParams p) {
  __shared__ __attribute__((aligned(16))) float p_lds[kDecWaves][TK];
  __shared__ float part[kDecWaves][E + 2];
  // K's transposition of an 8-bit append: by the one wave of the row's last tile.
  __shared__ __attribute__((aligned(16))) uint32_t kl[APPEND && F8 ? Store8Shape<E>::LDS_WORDS : 1];
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  const int64_t s = (uint32_t)row / (uint32_t)p.heads, h = row - s * p.heads;
  const int64_t tile = (int64_t)blockIdx.y * kDecWaves + wv;
  // For a host that polls it while the decode runs; nothing else has to be visible with it.
  // First of all, or behind the row's length, whichever costs less: an append N=1 H=32, window
  // 1023, 10.6 us against 10.9; without one, 8-bit N=64 H=32 194.5 us against 192.0.
  auto tell = [&]() __attribute__((always_inline)) {
    if (p.longest && (blockIdx.x | blockIdx.y) == 0 && wv == 0) {
      const int64_t longest = longest_of(p);
      if ((threadIdx.x & 63) == 0) __hip_atomic_store(p.longest, longest, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
  };
  if (APPEND) tell();
  const Span sp = span_of<APPEND && F8>(p, s);
  // Waves past the row's last tile exit (the barrier below waits for the others only).  A
  // row with no key has one tile of nothing, and is written as exactly 0.
  if (tile >= sp.tiles) return;
  if (!APPEND) tell();
  win_tile<E, BF, F8, APPEND, TK>(p, sp, s, h, tile, p_lds[wv], part[wv], kl);
  uint64_t seen = 0;
  if (p.counters && wv == 0) seen = __hip_atomic_load(p.counters + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (wv != 0) return;
  constexpr int DPC = E >= 64 ? E / 64 : 1;
  const int lane = threadIdx.x & 63;
  const int n = (int)min<int64_t>(kDecWaves, sp.tiles - (int64_t)blockIdx.y * kDecWaves);
  float mx, acc[DPC];
  const float l = merge_states<E, DPC>(n, [&](int t, int i) {
    return part[t][i == -1 ? E : (i == -2 ? E + 1 : i)];
  }, mx, acc);
  if (sp.tiles <= kDecWaves) {
    if (lane * DPC < E) store_out<DPC, BF>(p.out, row * E + lane * DPC, acc, l > 0.f ? 1.f / l : 0.f);
    return;
  }
  const int64_t slot = row * cdiv(p.tiles, kDecWaves) + blockIdx.y;
  if (p.counters) {
    merge_in_last_block<E, BF>(p, row, slot, (int)cdiv(sp.tiles, kDecWaves), seen, mx, l, acc, lane);
    return;
  }
  if (lane * DPC < E) {
#pragma unroll
    for (int i = 0; i < DPC; ++i) p.part_acc[slot * E + lane * DPC + i] = acc[i];
  }
  if (lane == 0) {
    p.part_ml[2 * slot] = mx;
    p.part_ml[2 * slot + 1] = l;
  }
}

// One wave per row of more than one block, where the rows' last blocks do not: merges the
// blocks' partials.
template <int E, bool BF, bool FOLD>
__global__ __launch_bounds__(256) void win_decode_combine_kernel(WinDecodeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= p.nseqs * p.heads) return;
  const int64_t tiles = span_of<FOLD>(p, row / p.heads).tiles;
  if (tiles <= kDecWaves) return;  // written by its block
  merge_partials<E, BF, false>(p, row, (int)cdiv(tiles, kDecWaves), lane);
}

// The most tiles that a row can have: its page table's capacity, or the units of the
// sinks and of a window that begins at any key of its first unit.  (FOLD: one more, for the
// last page's own tile.)
int64_t win_decode_tiles(int64_t pt_width, int64_t page, int64_t left, int64_t sinks) {
  int64_t units = pt_width * page / kUnit;
  if (left >= 0) {
    const int64_t seen = cdiv(sinks, kUnit) + cdiv(left + kUnit, kUnit);
    units = units < seen ? units : seen;
  }
  return cdiv(units, kWinTile / kUnit);
}

// The decode stores a new token itself for up to kFusedAppendMaxRows rows (as ca_decode), if
// the page of an 8-bit cache fits a tile.
bool win_decode_folds(int64_t rows, int64_t page, bool fp8) {
  return rows <= kFusedAppendMaxRows && (!fp8 || page <= kWinTile);
}

// Partial slots: one per (row, block of 8 tiles) when rows can outgrow one block.
int64_t win_decode_slots(int64_t rows, int64_t tiles) { return tiles > kDecWaves ? rows * cdiv(tiles, kDecWaves) : 0; }

template <int E, bool BF, bool F8>
static int win_decode_launch_t(const WinDecodeParams& p, hipStream_t stream) {
  const int64_t rows = p.nseqs * p.heads;
  const int64_t gy = p.tiles > kDecWaves ? cdiv(p.tiles, kDecWaves) : 1;
  if (rows > 0x7fffffff || p.page > 0x7fffffff || gy > 65535 || win_decode_slots(rows, p.tiles) > p.slots) return CA_DECLINED;
  const dim3 grid((unsigned)rows, (unsigned)gy), block(64 * kDecWaves);
  if (p.k_new)
    hipLaunchKernelGGL((win_decode_kernel<E, BF, F8, true, kWinTile>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((win_decode_kernel<E, BF, F8, false, kWinTile>), grid, block, 0, stream, p);
  const int st = ca_launch_status();
  if (st != CA_OK || gy == 1 || p.counters) return st;
  const dim3 cg((unsigned)cdiv(rows, 4));
  if (F8 && p.k_new)
    hipLaunchKernelGGL((win_decode_combine_kernel<E, BF, true>), cg, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((win_decode_combine_kernel<E, BF, false>), cg, dim3(256), 0, stream, p);
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
