// mcpm_logits.hip -- the rules on logits that come before sampling: penalties
// for ids of the history, biases, a mask of allowed ids (mcpm_process_logits).
//
//   c > 0:  l <- (l > 0 ? l / rep : l * rep) - (freq * c + pres)
//   listed: l <- l + bias;   not allowed: l <- -inf
//
// One work group per (sequence, tile of ids): it counts the history's ids that
// fall into its tile and finds the last bias entry of each in LDS (integer
// atomics, so no order of arrival changes a result), then passes once over the
// tile's logits.  No scratch in device memory and one launch.  The logits are
// asked for before the counting starts, so that they arrive meanwhile.
#include "mcpm_device.h"
#include "mcpm_paged.h"

namespace mcpm {

namespace {

constexpr int LG_T = 512;

// PER quads of ids a lane.  VEC: rows and tiles are 16-byte aligned.
template <int PER, bool VEC>
__global__ void __launch_bounds__(LG_T) k_process_logits(float* __restrict__ logits, const mcpm_logit_rules r) {
  constexpr int TILE = LG_T * 4 * PER;
  __shared__ __attribute__((aligned(16))) unsigned cnt[TILE];
  __shared__ __attribute__((aligned(16))) unsigned last[TILE];
  const int b = blockIdx.y, id0 = blockIdx.x * TILE, tid = threadIdx.x;
  const int n = min(TILE, r.vocab - id0);
  float* row = logits + b * r.stride + id0;
  f32x4 l[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int i = (p * LG_T + tid) * 4;
    if (VEC && i + 3 < n) {
      l[p] = *reinterpret_cast<const f32x4*>(row + i);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) l[p][k] = row[min(i + k, n - 1)];
    }
  }
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    reinterpret_cast<u32x4*>(cnt)[p * LG_T + tid] = u32x4{0, 0, 0, 0};
    reinterpret_cast<u32x4*>(last)[p * LG_T + tid] = u32x4{0, 0, 0, 0};
  }
  __syncthreads();
  if (r.history) {
    const int h0 = r.history_starts[b], h1 = r.history_starts[b + 1];
    for (int i0 = h0; i0 < h1; i0 += 8 * LG_T) {
      int id[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) id[k] = r.history[min(i0 + k * LG_T + tid, h1 - 1)];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const unsigned o = static_cast<unsigned>(id[k]) - static_cast<unsigned>(id0);
        if (i0 + k * LG_T + tid < h1 && o < static_cast<unsigned>(n)) atomicAdd(&cnt[o], 1u);
      }
    }
  }
  const int b0 = r.bias ? r.bias_starts[b] : 0;
  if (r.bias)
    for (int i = b0 + tid; i < r.bias_starts[b + 1]; i += LG_T) {
      const unsigned o = static_cast<unsigned>(r.bias_ids[i]) - static_cast<unsigned>(id0);
      if (o < static_cast<unsigned>(n)) atomicMax(&last[o], static_cast<unsigned>(i - b0) + 1);
    }
  __syncthreads();
  const float rep = r.repetition ? r.repetition[b] : 1.0f;
  const float pres = r.presence ? r.presence[b] : 0.0f, freq = r.frequency ? r.frequency[b] : 0.0f;
  const uint32_t* ok = r.allowed ? r.allowed + b * r.allowed_stride + id0 / 32 : nullptr;
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int i = (p * LG_T + tid) * 4;
    if (i >= n) break;
    const u32x4 c = reinterpret_cast<const u32x4*>(cnt)[p * LG_T + tid], e = reinterpret_cast<const u32x4*>(last)[p * LG_T + tid];
    const uint32_t bits = ok ? ok[i >> 5] >> (i & 31) : 15u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float x = l[p][k];
      if (c[k]) x = (x > 0.0f ? x / rep : x * rep) - (freq * static_cast<float>(c[k]) + pres);
      if (e[k]) x += r.bias[b0 + static_cast<int>(e[k]) - 1];
      if (!(bits >> k & 1)) x = -__builtin_inff();
      l[p][k] = x;
    }
    if (VEC && i + 3 < n) {
      *reinterpret_cast<f32x4*>(row + i) = l[p];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) row[i + k] = l[p][k];
    }
  }
}

template <int PER>
void process(float* logits, const mcpm_logit_rules& r, hipStream_t s) {
  const dim3 grid((r.vocab + LG_T * 4 * PER - 1) / (LG_T * 4 * PER), r.n_seq);
  if (reinterpret_cast<uintptr_t>(logits) % 16 == 0 && r.stride % 4 == 0)
    hipLaunchKernelGGL((k_process_logits<PER, true>), grid, dim3(LG_T), 0, s, logits, r);
  else
    hipLaunchKernelGGL((k_process_logits<PER, false>), grid, dim3(LG_T), 0, s, logits, r);
}

}  // namespace

// Every tile reads the whole history and holds 8 bytes of LDS an id, so tiles of
// 4096 ids run where there are work groups enough: 64 rows of 130,560 with 8192
// ids of history take 18.5 us with them (3.7 TB/s), 20.6 with 2048, 23 with 8192.
hipError_t launch_process_logits(float* logits, const mcpm_logit_rules& r, int n_cu, hipStream_t s) {
  if (static_cast<int64_t>(r.n_seq) * ((r.vocab + 4095) / 4096) >= 2 * n_cu) process<2>(logits, r, s);
  else process<1>(logits, r, s);
  return hipGetLastError();
}

}  // namespace mcpm
