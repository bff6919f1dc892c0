// What the paged decodes share: a row's output, the merge of a block's waves in LDS and
// the merge of a row's block partials (ca_decode.hip, ca_win_decode.hip).
#pragma once

#include "ca_device.h"
#include "ca_internal.h"

namespace ca {

constexpr int kDecWaves = 8;  // tiles (waves) per block

// out[idx .. idx+N) = v * inv in the output dtype (bf16: round to nearest even).
template <int N, bool BF>
__device__ __forceinline__ void store_out(void* out, int64_t idx, const float* v, float inv) {
  if constexpr (BF && N % 2 == 0) {
    uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(out) + idx);
#pragma unroll
    for (int i = 0; i < N; i += 2) o[i / 2] = pack_bf16x2(v[i] * inv, v[i + 1] * inv);
  } else if constexpr (BF) {
    uint16_t* o = reinterpret_cast<uint16_t*>(out) + idx;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (uint16_t)pack_bf16x2(v[i] * inv, 0.f);
  } else {
    float* o = reinterpret_cast<float*>(out) + idx;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = v[i] * inv;
  }
}

// Merges n partial states (m_t, l_t, acc_t) with weights 2^(m_t - M): lane-wise
// dims lane*DPC.., returns the merged sum; acc gets the merged P.V.
template <int E, int DPC, typename Get>
__device__ __forceinline__ float merge_states(int n, Get&& get, float& mx, float (&acc)[DPC]) {
  const int lane = threadIdx.x & 63;
  mx = -INFINITY;
  for (int t = 0; t < n; ++t) mx = fmaxf(mx, get(t, -1));
#pragma unroll
  for (int i = 0; i < DPC; ++i) acc[i] = 0.f;
  float l = 0.f;
  if (mx == -INFINITY) return 0.f;  // nothing readable
  for (int t = 0; t < n; ++t) {
    const float wgt = __builtin_amdgcn_exp2f(get(t, -1) - mx);
    l = fmaf(wgt, get(t, -2), l);
    if (lane * DPC < E) {
#pragma unroll
      for (int i = 0; i < DPC; ++i) acc[i] = fmaf(wgt, get(t, lane * DPC + i), acc[i]);
    }
  }
  return l;
}

// A partial-slot float: a plain load, or (COHERENT) a relaxed agent-scope atomic
// load, which reads the value the device-wide coherence point holds (the in-kernel
// merge reads partials other blocks, perhaps on other XCDs, wrote this launch).
template <bool COHERENT>
__device__ __forceinline__ float slot_load(float* q) {
  if constexpr (COHERENT) return __hip_atomic_load(q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return *q;
}

// Merges row `row`'s n block partials (slots row * nb .. + n - 1) and writes the
// row's output: one wave, lane l taking dims l * DPC ...  The partials are read C at
// a time, every load of a round issued before any is used (the merge is latency-
// bound: a row has a few KB of partials); rounds merge online.  A row of at most C
// blocks merges in one round, with the same arithmetic as a single pass (weights
// 2^(m_t - M) against the row's max M).
template <int E, bool BF, bool COHERENT>
__device__ __forceinline__ void merge_partials(const DecodeParams& p, int64_t row, int n, int lane) {
  constexpr int DPC = E >= 64 ? E / 64 : 1;
  constexpr int C = 8;
  const int64_t nb = cdiv(p.tiles, kDecWaves);
  const bool dims = lane * DPC < E;
  float* ml = p.part_ml + row * nb * 2;
  float* pa = p.part_acc + row * nb * E + (dims ? lane * DPC : 0);
  float m = -INFINITY, l = 0.f, acc[DPC];
#pragma unroll
  for (int i = 0; i < DPC; ++i) acc[i] = 0.f;
  for (int t0 = 0; t0 < n; t0 += C) {
    float mt[C], lt[C], at[C][DPC];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const bool in = t0 + c < n;
      mt[c] = in ? slot_load<COHERENT>(ml + 2 * (t0 + c)) : -INFINITY;
      lt[c] = in ? slot_load<COHERENT>(ml + 2 * (t0 + c) + 1) : 0.f;
#pragma unroll
      for (int i = 0; i < DPC; ++i) at[c][i] = in && dims ? slot_load<COHERENT>(pa + (int64_t)(t0 + c) * E + i) : 0.f;
    }
    float mc = m;
#pragma unroll
    for (int c = 0; c < C; ++c) mc = fmaxf(mc, mt[c]);
    if (mc == -INFINITY) continue;  // nothing readable yet
    const float sc = __builtin_amdgcn_exp2f(m - mc);  // 0 on the first readable round
    l *= sc;
#pragma unroll
    for (int i = 0; i < DPC; ++i) acc[i] *= sc;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float w = __builtin_amdgcn_exp2f(mt[c] - mc);
      l = fmaf(w, lt[c], l);
#pragma unroll
      for (int i = 0; i < DPC; ++i) acc[i] = fmaf(w, at[c][i], acc[i]);
    }
    m = mc;
  }
  if (dims) store_out<DPC, BF>(p.out, row * E + lane * DPC, acc, l > 0.f ? 1.f / l : 0.f);
}

}  // namespace ca
