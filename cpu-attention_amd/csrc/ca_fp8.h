// The 8-bit cache's store of one page (shared by ca_fp8.hip and the decode's append).
//
// The rule, for each page and head that a call puts tokens in.  With a the largest finite
// magnitude among those tokens' elements of the head,
//   need = the smallest 2^k, k >= -100, with a <= 448 * 2^k (448: e4m3's largest value);
//   a call that writes the page's position 0 starts the page anew: scale = need, and
//   what the page held is forgotten (its other codes stay, under a scale that is not
//   theirs); any other call keeps what it holds: scale = max(scale, need), and if that
//   grew, the page's codes become e4m3(code * old / scale);
//   each token's code is e4m3(x / scale), rounded to nearest even; inf and NaN are NaN
//   codes and take no part in a.
// Scales are powers of two, so dividing by them is exact and a value is rounded once;
// rescaling a code is exact too unless it becomes subnormal (below 2^-6, whose step then is
// 2^-18 of the page's largest value).  Growing is what lets a page be filled token by
// token without knowing what comes; pages are filled from position 0 on.
#pragma once

#include "ca_device.h"
#include "ca_internal.h"

namespace ca {

constexpr int kMinScaleExp = -100;
constexpr float kMinScale = 0x1p-100f;
// The smallest power of two from 2^-100 that takes magnitudes up to `top` (finite) to 448
// = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float top) {
  const uint32_t b = __float_as_uint(top);
  int k = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  k = k > kMinScaleExp ? k : kMinScaleExp;
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

// The larger of a and |x|, if x is finite.
__device__ __forceinline__ float max_finite(float a, float x) {
  const float y = fabsf(x);
  return fmaxf(a, y < INFINITY ? y : 0.f);
}

// Eight neighbouring elements of a row as they lie in memory, and as fp32.
template <bool BF>
struct Row8 {
  u32x4 w[BF ? 1 : 2];
  __device__ __forceinline__ void load(const void* src, int64_t i) {
    const char* at = reinterpret_cast<const char*>(src) + i * (BF ? 2 : 4);
#pragma unroll
    for (int k = 0; k < (BF ? 1 : 2); ++k) w[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at) + k);
  }
  __device__ __forceinline__ void widen(float (&x)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t v = BF ? w[0][k / 2] : w[BF ? 0 : k / 4][k % 4];
      x[k] = !BF ? __uint_as_float(v) : (k & 1 ? bf16_hi(v) : bf16_lo(v));
    }
  }
};

// n words of codes at `at` times `ratio`, by one wave.
__device__ __forceinline__ void rescale(uint32_t* at, int64_t words, float ratio, int lane) {
  for (int64_t i = 4 * lane; i < words; i += 4 * kWave) {
    u32x4 w = *reinterpret_cast<const u32x4*>(at + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t v = w[k];
      const f32x2 lo = e4m3_lo(v), hi = e4m3_hi(v);
      w[k] = e4m3_word(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
    }
    *reinterpret_cast<u32x4*>(at + i) = w;
  }
}

template <int E>
struct Store8Shape {
  static constexpr int W = E / 4;          // words per row of codes
  static constexpr int LPR = E / 8;        // lanes per row
  static constexpr int RPL = kWave / LPR;  // rows per load
  static constexpr int NL = 16 / RPL;      // loads of 16 positions
  static constexpr int LD = 20;            // LDS words per K word row (16 positions, padded)
  static constexpr int LDS_WORDS = W * LD;
};

// Puts the tokens of (blk, h) into the cache: token_of(t) names position t's token, or is
// negative.  One wave; kl is its LDS_WORDS words of LDS.
template <int E, bool BF, typename F>
__device__ __forceinline__ void store_page(const Store8Page& p, int64_t blk, int64_t h, uint32_t* kl, F&& token_of) {
  using D = Store8Shape<E>;
  constexpr int W = D::W, LPR = D::LPR, RPL = D::RPL, NL = D::NL, LD = D::LD;
  const int lane = threadIdx.x & 63, r = lane / LPR, dl = lane % LPR;
  const int64_t bh = blk * p.heads + h;
  uint32_t* kw = p.kc + bh * p.page * W;
  uint32_t* vw = p.vc + bh * p.page * W;
  Row8<BF> kx[NL], vx[NL];
  int tok[NL];
  // The tokens of positions t0 .. t0 + 15 and their rows; whether there are any.
  auto load = [&](int64_t t0) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      tok[i] = token_of(t0 + i * RPL + r);
      any |= tok[i] >= 0;
    }
    if (!__any(any)) return false;
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (tok[i] >= 0) {
        const int64_t at = (int64_t)tok[i] * p.tok_stride + h * E + 8 * dl;
        kx[i].load(p.key, at);
        vx[i].load(p.value, at);
      }
    return true;
  };
  // The maxima, over every 16 positions of the page.  The last ones looked at stay in
  // registers: all there is in a page of 16, others are read again below.
  float mk = 0.f, mv = 0.f;
  bool found = false, anew = false;
  for (int64_t t0 = 0; t0 < p.page; t0 += 16) {
    if (!load(t0)) continue;
    found = true;
    if (t0 == 0) anew = __any(r == 0 && tok[0] >= 0);
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (tok[i] >= 0) {
        float x[8];
        kx[i].widen(x);
#pragma unroll
        for (int j = 0; j < 8; ++j) mk = max_finite(mk, x[j]);
        vx[i].widen(x);
#pragma unroll
        for (int j = 0; j < 8; ++j) mv = max_finite(mv, x[j]);
      }
  }
  if (!found) return;
  float ks = scale_for(wave_max(mk)), vs = scale_for(wave_max(mv));
  if (!anew) {
    const float ko = p.k_scale[bh], vo = p.v_scale[bh];
    const float k0 = ko >= kMinScale ? ko : kMinScale, v0 = vo >= kMinScale ? vo : kMinScale;
    if (ks > k0) rescale(kw, p.page * W, k0 / ks, lane);
    if (vs > v0) rescale(vw, p.page * W, v0 / vs, lane);
    ks = fmaxf(ks, k0);
    vs = fmaxf(vs, v0);
    // The tokens' words go over rescaled ones that other lanes wrote.
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  }
  const float ki = 1.f / ks, vi = 1.f / vs;
  const int64_t last = p.page - 16;
  for (int64_t t0 = last; t0 >= 0; t0 -= 16) {
    if (last > 0 && !load(t0)) continue;
    uint32_t own = 0;  // positions of the 16 that get a token
    wave_lds_sync();   // the reads of the 16 before
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const uint64_t b = __ballot(tok[i] >= 0);
#pragma unroll
      for (int k = 0; k < RPL; ++k) own |= (uint32_t)(b >> (k * LPR) & 1) << (i * RPL + k);
      if (tok[i] >= 0) {
        const int t = i * RPL + r;
        float k[8], v[8];
        kx[i].widen(k);
        vx[i].widen(v);
        kl[(2 * dl) * LD + t] = e4m3_word(k[0] * ki, k[1] * ki, k[2] * ki, k[3] * ki);
        kl[(2 * dl + 1) * LD + t] = e4m3_word(k[4] * ki, k[5] * ki, k[6] * ki, k[7] * ki);
        const u32x2 vq = {e4m3_word(v[0] * vi, v[1] * vi, v[2] * vi, v[3] * vi),
                          e4m3_word(v[4] * vi, v[5] * vi, v[6] * vi, v[7] * vi)};
        __builtin_nontemporal_store(vq, reinterpret_cast<u32x2*>(vw + (t0 + t) * W + 2 * dl));
      }
    }
    wave_lds_sync();
#pragma unroll
    for (int x = lane; x < 4 * W; x += kWave) {
      const int w = x >> 2, tq = x & 3;
      const uint32_t mine = own >> (4 * tq) & 15u;
      const u32x4 q = *reinterpret_cast<const u32x4*>(kl + w * LD + 4 * tq);
      uint32_t* to = kw + w * p.page + t0 + 4 * tq;
      if (mine == 15u) {
        *reinterpret_cast<u32x4*>(to) = q;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (mine >> j & 1) to[j] = q[j];
      }
    }
  }
  if (lane == 0) {
    p.k_scale[bh] = ks;
    p.v_scale[bh] = vs;
  }
}

}  // namespace ca
