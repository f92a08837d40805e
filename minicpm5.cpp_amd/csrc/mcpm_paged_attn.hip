// mcpm_paged_attn.hip -- attention over the paged cache.
//
//   s_j = scale * q.k_j;  cap: c tanh(s/c);  - slope |i - j|;  seen: see mcpm_attn_rules
//   o = sum_j p_j v_j,  p_j = exp(s_j - m) / z over the seen j;  weight_j += p_j
//
// Scores are held in units of log2.
#include <algorithm>

#include "mcpm_paged_score.h"

namespace mcpm {

namespace {

// ---------------------------------------------------------------- few rows --
// A row block is up to 16 rows (new tokens x the kv head's query heads, token
// by token).  A wave takes 32 positions at a time and forms the transposed
// products S^T = K Q^T and O^T = V^T P^T on the 16-row matrix instructions, so
// a lane's column is one row all the way: of the 32 positions the lane with
// row n and lane group g holds p0 + 4g + i and p0 + 16 + 4g + i (i < 4), as
// many as the second product wants of it, and any order of the positions will
// do there as long as V's operand has the same.  K comes from memory straight in
// operand order (a lane: 16 bytes of one position), V as whole rows (a lane: 16
// bytes of each of its 8 positions), turned by byte permutes within the lane.
// Nothing passes through LDS but the page offsets and, at the end, the waves'
// partial outputs.

constexpr int FEW_ROWS = 16;
constexpr int FEW_STEP = 32;                // positions of a wave's step
constexpr int FEW_ROUND = 4 * FEW_STEP;     // of a work group's
constexpr int FEW_MIN_CHUNK = 256;
constexpr int FEW_TARGET = 4;               // work groups per CU
constexpr int FEW_MOST = 32;                // new tokens x group up to which these kernels run
constexpr int FEW_MAX_CHUNK = 2048;         // positions of a work group, at most

struct FewArgs {
  PagedView kv;
  BatchView bt;
  RuleView rl;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  int n_heads, group, n_blocks;  // query heads per kv head; row blocks per (sequence, kv head)
  int chunk, n_splits;
  float* part_o;    // [seq][new token][head][split][hd], unnormalised
  float2* part_mz;  // [seq][new token][head][split]
  float* scores;    // [seq][kv head][row of the sequence][score_len], or null
  int score_len, score_rows;
};

__device__ __forceinline__ int64_t few_part(const FewArgs& a, int b, int t, int head, int split) {
  return ((static_cast<int64_t>(b) * a.bt.max_new + t) * a.n_heads + head) * a.n_splits + split;
}

// The positions of a row block.
struct FewBlock {
  int r_end;  // rows of the sequence
  int pos0;   // position of row 0 of the sequence
  KeyRange keys;
};
__device__ __forceinline__ FewBlock few_block(const FewArgs& a, int b, int rb, const SeqRows& sr, int len) {
  const int pos0 = len - sr.given, r_end = sr.n * a.group;
  const int t0 = rb * FEW_ROWS / a.group, t1 = (min(rb * FEW_ROWS + FEW_ROWS, r_end) - 1) / a.group;
  return FewBlock{r_end, pos0, key_range(a.rl, b, pos0 + t0, pos0 + t1, len)};
}

// Page offsets of a chunk (a page outside the pool stands at the first one, to be masked);
// whether all of this lane's are in the pool.
__device__ __forceinline__ bool load_page_offsets(const BatchView& bt, const PagedView& kv, int b, int c0, int c1, int64_t* s_off) {
  bool ok = true;
  const int first = c0 >> kv.page_shift, n = ((c1 - 1) >> kv.page_shift) - first + 1;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int page = page_of(bt, kv, b, (first + i) << kv.page_shift);
    s_off[i] = page < 0 ? 0 : page * kv.page_stride;
    ok = ok && page >= 0;
  }
  return ok;
}

// The plain computation of one row over positions [c0, c1), by the whole work
// group, for values that the matrix products cannot keep apart: a share of 0
// times what a masked place holds.  Returns this lane's element tid of sum
// p v, and (m, z).
template <typename TC, typename TI>
__device__ __forceinline__ float exact_row(const FewArgs& a, int b, int kh, int row, int head, int pos, int c0, int c1, float* s_q,
                                        float* s_p, float* s_red, float2* mz) {
  const PagedView& kv = a.kv;
  const int tid = threadIdx.x, hd = kv.hd;
  __syncthreads();
  if (tid < hd) s_q[tid] = static_cast<float>(static_cast<const TI*>(a.q)[row * a.q_stride + head * hd + tid]);
  __syncthreads();
  const ScoreRule sr = score_rule(a.rl);
  const RowRule rr = row_rule(a.rl, b, pos);
  const float slope = a.rl.slopes ? a.rl.slopes[head] * LOG2E : 0.0f;
  float m = MAX_START, z = 0.0f, o = 0.0f;
  for (int j0 = c0; j0 < c1; j0 += 256) {
    const int j = j0 + tid;
    float s = -__builtin_inff();
    const int page = j < c1 && pos >= 0 && seen(a.rl, rr, b, j) ? page_of(a.bt, kv, b, j) : -1;
    if (page >= 0) {
      const TC* k = reinterpret_cast<const TC*>(kv.k) + elem_of(kv, page, j, kh);
      float d = 0.0f;
      for (int i = 0; i < hd; ++i) d = __builtin_fmaf(s_q[i], static_cast<float>(k[i]), d);
      s = score_of(sr, d, sr.mul) - slope * fabsf(static_cast<float>(pos - j));
    }
    float w = wave_max(s);
    if ((tid & 63) == 0) s_red[tid >> 6] = w;
    __syncthreads();
    w = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float mn = fmaxf(m, w), scale = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    s_p[tid] = __builtin_amdgcn_exp2f(s - m);
    __syncthreads();
    z *= scale;
    o *= scale;
    for (int i = 0; i < min(256, c1 - j0); ++i) {
      const float p = s_p[i];
      if (p == 0.0f) continue;
      z += p;
      if (tid < hd) {
        const int pg = page_of(a.bt, kv, b, j0 + i);  // p != 0: in the pool
        if (pg >= 0) o = __builtin_fmaf(p, static_cast<float>((reinterpret_cast<const TC*>(kv.v) + elem_of(kv, pg, j0 + i, kh))[tid]), o);
      }
    }
    __syncthreads();
  }
  *mz = make_float2(m, z);
  return o;
}

template <typename TC, typename TI, int DP>
struct FewTile;

// 16-bit caches.
template <typename TC, typename TI, int DP>
struct FewTile16 {
  typedef typename Half<TC>::V8 V8;
  static constexpr int NT = Terms<TC, TI>::N;
  static constexpr int KS = DP / 32;                 // K operand loads of a tile
  static constexpr int VW = DP >= 128 ? 8 : DP / 16; // elements of a V load
  static constexpr int VH = DP / (16 * VW);          // V loads of a row
  static constexpr int NO = DP / 16;                 // output tiles
  V8 q[NT][KS];
  f32x4 o[NO];
  float mul;  // raw product to score
  union VRow {
    uint32_t w[VW / 2];
    u32x4 w4;
    u32x2 w2;
  };
  V8 k[2][KS];
  VRow v[8][VH];

  // Rows of 32 bits over halves are brought to a top exponent of 8 by a power of
  // two, so that neither term leaves a half's range; products take it back.
  __device__ __forceinline__ void load_q(const TI* row, int hd, float score_mul) {
    const int g = (threadIdx.x >> 4) & 3;
    float x[KS][8];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = 32 * s + 8 * g;
        x[s][i] = row && d < hd ? static_cast<float>(row[d + i]) : 0.0f;
        top = fmaxf(top, fabsf(x[s][i]));
      }
    mul = score_mul;
    if (NT == 2) {
      top = fmaxf(top, lane_xor16(top));
      top = fmaxf(top, lane_xor32(top));
      if (top > 0.0f && top < __builtin_inff()) {
        const int e = 9 - __builtin_amdgcn_frexp_expf(top);
        mul = ldexpf(score_mul, -e);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[s][i] = ldexpf(x[s][i], e);
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      V8 t[NT];
      split_terms<TC, NT>(x[s], t);
#pragma unroll
      for (int n = 0; n < NT; ++n) q[n][s] = t[n];
    }
#pragma unroll
    for (int j = 0; j < NO; ++j) o[j] = f32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void load_k(int t, const TC* row, int hd) {
    const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int s = 0; s < KS; ++s) k[t][s] = *reinterpret_cast<const V8*>(row + min(32 * s + 8 * g, hd - 8));
  }
  __device__ __forceinline__ void load_v(int i, const TC* row, int hd) {
    const int m = threadIdx.x & 15;
#pragma unroll
    for (int h = 0; h < VH; ++h) {
      const TC* p = row + min(16 * VW * h + VW * m, hd - VW);
      if constexpr (VW == 8) v[i][h].w4 = *reinterpret_cast<const u32x4*>(p);
      else v[i][h].w2 = *reinterpret_cast<const u32x2*>(p);
    }
  }
  __device__ __forceinline__ f32x4 scores(int t) {
    f32x4 s{0, 0, 0, 0};
#pragma unroll
    for (int n = NT - 1; n >= 0; --n)
#pragma unroll
      for (int i = 0; i < KS; ++i) s = Half<TC>::mma16(k[t][i], q[n][i], s);
    return s;
  }
  __device__ __forceinline__ void add(const float (&p)[8]) {
    V8 t[NT];
    split_terms<TC, NT>(p, t);
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int w = 0; w < VW / 2; ++w) {
        u32x4 lo, hi;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          lo[r] = __builtin_amdgcn_perm(v[2 * r + 1][h].w[w], v[2 * r][h].w[w], 0x05040100u);
          hi[r] = __builtin_amdgcn_perm(v[2 * r + 1][h].w[w], v[2 * r][h].w[w], 0x07060302u);
        }
        const V8 a0 = __builtin_bit_cast(V8, lo), a1 = __builtin_bit_cast(V8, hi);
        const int j = h * VW + 2 * w;
#pragma unroll
        for (int n = NT - 1; n >= 0; --n) {
          o[j] = Half<TC>::mma16(a0, t[n], o[j]);
          o[j + 1] = Half<TC>::mma16(a1, t[n], o[j + 1]);
        }
      }
  }
  // Output element of tile j at the lane's index i.
  static __device__ __forceinline__ int d_of(int j, int i) {
    const int g = (threadIdx.x >> 4) & 3;
    return 16 * VW * (j / VW) + VW * (4 * g + i) + j % VW;
  }
};
template <typename TI, int DP>
struct FewTile<_Float16, TI, DP> : FewTile16<_Float16, TI, DP> {};
template <typename TI, int DP>
struct FewTile<__bf16, TI, DP> : FewTile16<__bf16, TI, DP> {};

// 32-bit caches: v_mfma_f32_16x16x4_f32, whose K operand takes one element of
// each of 4 lane groups: element c of the 16 bytes that a lane loads goes into
// instruction c.  V needs no turning.
template <int DP>
struct FewTile<float, float, DP> {
  static constexpr int KS = DP / 16, VH = DP / 64, NO = DP / 16;
  f32x4 q[KS], o[NO], k[2][KS], v[8][VH];
  float mul;
  __device__ __forceinline__ void load_q(const float* row, int hd, float score_mul) {
    const int g = (threadIdx.x >> 4) & 3;
    mul = score_mul;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 4 * g;
      q[s] = row && d < hd ? *reinterpret_cast<const f32x4*>(row + d) : f32x4{0, 0, 0, 0};
      o[s] = f32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void load_k(int t, const float* row, int hd) {
    const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int s = 0; s < KS; ++s) k[t][s] = *reinterpret_cast<const f32x4*>(row + min(16 * s + 4 * g, hd - 4));
  }
  __device__ __forceinline__ void load_v(int i, const float* row, int hd) {
    const int m = threadIdx.x & 15;
#pragma unroll
    for (int h = 0; h < VH; ++h) v[i][h] = *reinterpret_cast<const f32x4*>(row + min(64 * h + 4 * m, hd - 4));
  }
  __device__ __forceinline__ f32x4 scores(int t) {
    f32x4 s{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][i][c], q[i][c], s, 0, 0, 0);
    return s;
  }
  __device__ __forceinline__ void add(const float (&p)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int h = 0; h < VH; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[4 * h + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][h][c], p[i], o[4 * h + c], 0, 0, 0);
  }
  static __device__ __forceinline__ int d_of(int j, int i) {
    const int g = (threadIdx.x >> 4) & 3;
    return 64 * (j / 4) + 4 * (4 * g + i) + j % 4;
  }
};

template <typename TC, typename TI, int DP>
__global__ void __launch_bounds__(256) k_attention_few(const FewArgs a) {
  __shared__ __attribute__((aligned(16))) float s_o[4][FEW_ROWS][DP + 4];
  __shared__ float s_m[4][FEW_ROWS], s_z[4][FEW_ROWS];
  __shared__ int s_bad;
  extern __shared__ int64_t s_off[];
  const PagedView& kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, n16 = lane & 15, g = lane >> 4;
  const int b = blockIdx.y;
  const int per = kv.n_kv_heads * a.n_blocks;
  const int split = blockIdx.x / per, kh = blockIdx.x % per % kv.n_kv_heads, rb = blockIdx.x % per / kv.n_kv_heads;
  const SeqRows sr = seq_rows(a.bt, b);
  const int len = seq_len(a.bt, kv, b);
  if (rb * FEW_ROWS >= sr.n * a.group) return;
  const FewBlock fb = few_block(a, b, rb, sr, len);
  const int c0 = fb.keys.lo + split * a.chunk, c1 = min(fb.keys.hi, c0 + a.chunk);
  if (split && c0 >= fb.keys.hi) return;  // the first one answers for rows that see nothing

  const int r = rb * FEW_ROWS + n16;
  const bool row_in = r < fb.r_end;
  const int t = row_in ? r / a.group : 0, head = kh * a.group + (row_in ? r - t * a.group : 0);
  const int64_t row = sr.r0 + t;
  const int pos = fb.pos0 + t;
  const ScoreRule rule = score_rule(a.rl);
  const RowRule rr = row_rule(a.rl, b, row_in ? pos : -1);
  const float slope = a.rl.slopes ? a.rl.slopes[head] * LOG2E : 0.0f;
  const TC* kc = reinterpret_cast<const TC*>(kv.k) + kh * kv.head_stride;
  const TC* vc = reinterpret_cast<const TC*>(kv.v) + kh * kv.head_stride;
  float* sc_row = a.scores && row_in ? a.scores + ((static_cast<int64_t>(b) * kv.n_kv_heads + kh) * a.score_rows + r) * a.score_len : nullptr;

  const bool ok = c0 < c1 ? load_page_offsets(a.bt, kv, b, c0, c1, s_off) : true;
  const bool bad_pages = __syncthreads_or(!ok);
  const int first_page = c0 >> kv.page_shift;
  // element offset of a position's row, of kv head 0; past the chunk's end the last one
  auto offset = [&](int j) -> int64_t {
    j = min(j, c1 - 1);
    return s_off[(j >> kv.page_shift) - first_page] +
           static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(j & kv.page_mask)) * static_cast<uint32_t>(kv.pos_stride));
  };

  FewTile<TC, TI, DP> tile;
  tile.load_q(row_in && pos >= 0 ? static_cast<const TI*>(a.q) + row * a.q_stride + head * kv.hd : nullptr, kv.hd, rule.mul);

  constexpr float LIFT = __is_same(TC, _Float16) ? 15.0f : 0.0f;
  float m = MAX_START, z = 0.0f;
  // Rows of one block differ in position by up to 15 tokens: a step that lies
  // before all of them and inside every window needs no masks.
  const int pos_min = fb.pos0 + rb * FEW_ROWS / a.group, pos_max = fb.pos0 + (min(rb * FEW_ROWS + FEW_ROWS, fb.r_end) - 1) / a.group;
  const bool plain = !a.rl.docs && !bad_pages && pos_min >= 0;
  for (int p0 = c0 + wv * FEW_STEP; p0 < c1; p0 += FEW_ROUND) {
#pragma unroll
    for (int T = 0; T < 2; ++T) tile.load_k(T, kc + offset(p0 + 16 * T + n16), kv.hd);
#pragma unroll
    for (int i = 0; i < 8; ++i) tile.load_v(i, vc + offset(p0 + 16 * (i >> 2) + 4 * g + (i & 3)), kv.hd);
    float s[8];
#pragma unroll
    for (int T = 0; T < 2; ++T) {
      const f32x4 x = tile.scores(T);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * T + i] = score_of(rule, x[i], tile.mul);
    }
    if (a.rl.slopes) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] -= slope * fabsf(static_cast<float>(pos - (p0 + 16 * (i >> 2) + 4 * g + (i & 3))));
    }
    if (!plain || p0 + FEW_STEP - 1 > pos_min || p0 + FEW_STEP > c1 || (a.rl.window > 0 && pos_max - p0 >= a.rl.window)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = p0 + 16 * (i >> 2) + 4 * g + (i & 3);
        const int jc = min(j, c1 - 1);
        bool ok = (j < c1) & seen(a.rl, rr, b, jc);
        if (bad_pages) ok &= page_of(a.bt, kv, b, jc) >= 0;
        s[i] = ok ? s[i] : -__builtin_inff();
      }
    }
    if (sc_row) {
      *reinterpret_cast<f32x4*>(sc_row + p0 + 4 * g) = f32x4{s[0], s[1], s[2], s[3]};
      *reinterpret_cast<f32x4*>(sc_row + p0 + 16 + 4 * g) = f32x4{s[4], s[5], s[6], s[7]};
    }
    // over halves the shares are taken against 2^-15 of the largest: what is
    // down to 2^-29 of it then stays a normal half
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7]))) - LIFT;
    if (__any(top > m)) {
      top = fmaxf(top, lane_xor16(top));
      top = fmaxf(top, lane_xor32(top));
      const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      z *= f;
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) tile.o[j] *= f;
    }
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(s[i] - m);
      z += p[i];
    }
    tile.add(p);
  }

  // the waves' partials, joined in LDS
  z += lane_xor16(z);
  z += lane_xor32(z);
  if (g == 0) {
    s_m[wv][n16] = m;
    s_z[wv][n16] = z;
  }
#pragma unroll
  for (int j = 0; j < DP / 16; j += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(&s_o[wv][n16][tile.d_of(j, i)]) = f32x4{tile.o[j][i], tile.o[j + 1][i], tile.o[j + 2][i], tile.o[j + 3][i]};
  if (tid == 0) s_bad = 0;
  __syncthreads();
  constexpr int TR = 256 / FEW_ROWS;  // lanes of a row here
  const int rn = tid / TR, part = tid % TR;
  const int rj = rb * FEW_ROWS + rn;
  const bool in = rj < fb.r_end;
  const int tj = in ? rj / a.group : 0, hj = kh * a.group + (in ? rj - tj * a.group : 0);
  const float M = fmaxf(fmaxf(s_m[0][rn], s_m[1][rn]), fmaxf(s_m[2][rn], s_m[3][rn]));
  float w[4], Z = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = __builtin_amdgcn_exp2f(s_m[i][rn] - M);
    Z += w[i] * s_z[i][rn];
  }
  const int64_t rowj = sr.r0 + tj;
  const int64_t at = few_part(a, b, tj, hj, split);
  const bool final = a.n_splits == 1;
  const float inv = Z == 0.0f ? 0.0f : 1.0f / Z;
  TI* dst = static_cast<TI*>(a.out) + rowj * a.out_stride + hj * kv.hd;
  bool bad = !(Z < __builtin_inff());
#pragma unroll
  for (int d0 = 0; d0 < DP; d0 += TR * 4) {
    const int d = d0 + part * 4;
    f32x4 acc{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) acc += w[i] * *reinterpret_cast<const f32x4*>(&s_o[i][rn][d]);
    if (d < kv.hd && in) {
      const float e = (acc[0] - acc[0]) + (acc[1] - acc[1]) + (acc[2] - acc[2]) + (acc[3] - acc[3]);
      bad = bad || e != 0.0f;
      if (final) {
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[d + i] = static_cast<TI>(acc[i] * inv);
      } else {
        *reinterpret_cast<f32x4*>(a.part_o + at * kv.hd + d) = acc;
      }
    }
  }
  if (in && part == 0 && a.part_mz) a.part_mz[at] = make_float2(M, Z);
  if (in && bad) s_bad = 1;
  __syncthreads();
  if (!s_bad) return;
  // Something infinite or NaN came up: perhaps only a share of 0 times it.
  for (int i = 0; i < FEW_ROWS && rb * FEW_ROWS + i < fb.r_end; ++i) {
    const int ri = rb * FEW_ROWS + i, ti = ri / a.group, hi = kh * a.group + ri - ti * a.group;
    float2 mz;
    const float o = exact_row<TC, TI>(a, b, kh, sr.r0 + ti, hi, fb.pos0 + ti, c0, c1, &s_o[0][0][0], &s_o[2][0][0], &s_m[0][0], &mz);
    const int64_t ai = few_part(a, b, ti, hi, split);
    if (tid < kv.hd) {
      if (final) static_cast<TI*>(a.out)[(sr.r0 + ti) * a.out_stride + hi * kv.hd + tid] = static_cast<TI>(mz.y == 0.0f ? 0.0f : o / mz.y);
      else a.part_o[ai * kv.hd + tid] = o;
    }
    if (tid == 0 && a.part_mz) a.part_mz[ai] = mz;
  }
}

// The splits' maxima and sums of a row joined, by a wave.
__device__ __forceinline__ float2 join_mz(const float2* mz, int n) {
  const int lane = threadIdx.x & 63;
  float M = MAX_START;
  for (int i = lane; i < n; i += 64) M = fmaxf(M, mz[i].x);
  M = wave_max(M);
  float Z = 0.0f;
  for (int i = lane; i < n; i += 64) Z += mz[i].y * __builtin_amdgcn_exp2f(mz[i].x - M);
  for (int s = 32; s; s >>= 1) Z += __shfl_xor(Z, s);
  return make_float2(M, Z);
}
__device__ __forceinline__ int active_splits(const FewArgs& a, const KeyRange& k) {
  return k.hi > k.lo ? (k.hi - k.lo + a.chunk - 1) / a.chunk : 1;
}

// A work group per (new token, head): the splits' partials into the output,
// 256 / (DP/4) of them at a time.
template <typename TI, int DP>
__global__ void __launch_bounds__(256) k_attention_join(const FewArgs a) {
  constexpr int LP = DP / 4, GR = 256 / LP;
  __shared__ f32x4 s_acc[GR][LP];
  const int b = blockIdx.y, tid = threadIdx.x, hd = a.kv.hd;
  const SeqRows sr = seq_rows(a.bt, b);
  const int t = blockIdx.x / a.n_heads, head = blockIdx.x % a.n_heads;
  if (t >= sr.n) return;
  const int rb = (t * a.group + head % a.group) / FEW_ROWS;
  const FewBlock fb = few_block(a, b, rb, sr, seq_len(a.bt, a.kv, b));
  const int n = active_splits(a, fb.keys);
  const int64_t at = few_part(a, b, t, head, 0);
  const float2 mz = join_mz(a.part_mz + at, n);
  const int d = tid % LP * 4;
  f32x4 acc{0, 0, 0, 0};
  if (d < hd)
    for (int i = tid / LP; i < n; i += GR) {
      const float2 x = a.part_mz[at + i];
      if (x.y != 0.0f) acc += __builtin_amdgcn_exp2f(x.x - mz.x) * *reinterpret_cast<const f32x4*>(a.part_o + (at + i) * hd + d);
    }
  s_acc[tid / LP][tid % LP] = acc;
  __syncthreads();
  if (tid >= LP || d >= hd) return;
  for (int i = 1; i < GR; ++i) acc += s_acc[i][tid];
  const float inv = mz.y == 0.0f ? 0.0f : 1.0f / mz.y;
  TI* dst = static_cast<TI*>(a.out) + (sr.r0 + t) * a.out_stride + head * hd + d;
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[i] = static_cast<TI>(acc[i] * inv);
}

// The positions' weights from the scores: a lane per position sums its rows in order.
__global__ void __launch_bounds__(256) k_attention_weight(const FewArgs a) {
  __shared__ float2 s_mz[FEW_ROWS];
  const int kh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, j = blockIdx.x * 256 + tid;
  const int len = seq_len(a.bt, a.kv, b);
  if (static_cast<int>(blockIdx.x) * 256 >= len) return;
  const SeqRows sr = seq_rows(a.bt, b);
  const int rows = sr.n * a.group;
  const float* sc = a.scores + (static_cast<int64_t>(b) * a.kv.n_kv_heads + kh) * a.score_rows * a.score_len + j;
  float sum = 0.0f;
  for (int r0 = 0; r0 < rows; r0 += FEW_ROWS) {
    const FewBlock fb = few_block(a, b, r0 / FEW_ROWS, sr, len);
    __syncthreads();
    for (int i = tid >> 6; i < FEW_ROWS && r0 + i < rows; i += 4) {
      const int t = (r0 + i) / a.group;
      const float2 mz = join_mz(a.part_mz + few_part(a, b, t, kh * a.group + r0 + i - t * a.group, 0), active_splits(a, fb.keys));
      if ((tid & 63) == 0) s_mz[i] = make_float2(mz.x, mz.y == 0.0f ? 0.0f : 1.0f / mz.y);
    }
    __syncthreads();
    if (j >= fb.keys.lo && j < fb.keys.hi)
      for (int i = 0; i < FEW_ROWS && r0 + i < rows; ++i)
        sum += __builtin_amdgcn_exp2f(sc[static_cast<int64_t>(r0 + i) * a.score_len] - s_mz[i].x) * s_mz[i].y;
  }
  if (j >= len) return;
  const int page = page_of(a.bt, a.kv, b, j);
  if (page >= 0) *weight_of(a.kv, page, j, kh) += sum;
}

__device__ __forceinline__ float simple_score(const RuleView& rl, float slope, float dot, int pos, int j) {
  const ScoreRule r = score_rule(rl);
  return score_of(r, dot, r.mul) - slope * LOG2E * fabsf(static_cast<float>(pos - j));
}

template <typename TC>
__device__ __forceinline__ float dot_row(const float* q, const TC* k, int hd) {
  float a = 0.0f;
  for (int d = 0; d < hd; ++d) a = __builtin_fmaf(q[d], static_cast<float>(k[d]), a);
  return a;
}

// One work group per (new token, query head): 256 positions at a time, a lane
// each for the scores, then a lane per output element for the sum over v.
template <typename TC, typename TI>
__global__ void __launch_bounds__(256) k_paged_attention(PagedView kv, BatchView bt, RuleView rl, TI* __restrict__ out,
                                                         int64_t out_stride, const TI* __restrict__ q, int64_t q_stride,
                                                         int n_heads, float2* __restrict__ mz) {
  __shared__ float s_q[PAGED_MAX_HD], s_p[256], s_red[4];
  const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, hd = kv.hd;
  const SeqRows sr = seq_rows(bt, b);
  if (t >= sr.n) return;
  const int row = sr.r0 + t, len = seq_len(bt, kv, b), pos = len - sr.given + t;
  const int kh = h / (n_heads / kv.n_kv_heads);
  if (tid < hd) s_q[tid] = static_cast<float>(q[row * q_stride + h * hd + tid]);
  __syncthreads();
  float m = MAX_START, z = 0.0f, o = 0.0f;
  if (pos >= 0) {
    const RowRule rr = row_rule(rl, b, pos);
    const float slope = rl.slopes ? rl.slopes[h] : 0.0f;
    for (int j0 = 0; j0 < len; j0 += 256) {
      const int j = j0 + tid;
      float s = -__builtin_inff();
      if (j < len && seen(rl, rr, b, j)) {
        const int page = page_of(bt, kv, b, j);
        if (page >= 0)
          s = simple_score(rl, slope, dot_row(s_q, reinterpret_cast<const TC*>(kv.k) + elem_of(kv, page, j, kh), hd), pos, j);
      }
      float w = wave_max(s);
      if ((tid & 63) == 0) s_red[tid >> 6] = w;
      __syncthreads();
      w = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
      const float mn = fmaxf(m, w);
      {
        const float scale = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        s_p[tid] = __builtin_amdgcn_exp2f(s - m);
        __syncthreads();
        z *= scale;
        o *= scale;
        for (int i = 0; i < min(256, len - j0); ++i) {
          const float p = s_p[i];
          if (p == 0.0f) continue;
          z += p;
          if (tid < hd) {
            const int page = page_of(bt, kv, b, j0 + i);
            o = __builtin_fmaf(p, static_cast<float>((reinterpret_cast<const TC*>(kv.v) + elem_of(kv, page, j0 + i, kh))[tid]), o);
          }
        }
      }
      __syncthreads();
    }
  }
  if (tid < hd) out[row * out_stride + h * hd + tid] = static_cast<TI>(z == 0.0f ? 0.0f : o / z);
  if (mz && tid == 0) mz[static_cast<int64_t>(row) * n_heads + h] = make_float2(m, z);
}

// weight of a position: a lane sums its shares over the rows and heads, in order.
template <typename TC, typename TI>
__global__ void __launch_bounds__(256) k_paged_weight(PagedView kv, BatchView bt, RuleView rl, const TI* __restrict__ q,
                                                      int64_t q_stride, int n_heads, const float2* __restrict__ mz) {
  const int j = blockIdx.x * 256 + threadIdx.x, kh = blockIdx.y, b = blockIdx.z, hd = kv.hd;
  const int len = seq_len(bt, kv, b), G = n_heads / kv.n_kv_heads;
  const SeqRows sr = seq_rows(bt, b);
  if (j >= len) return;
  const int page = page_of(bt, kv, b, j);
  if (page < 0) return;
  const TC* k = reinterpret_cast<const TC*>(kv.k) + elem_of(kv, page, j, kh);
  float sum = 0.0f;
  for (int t = 0; t < sr.n; ++t) {
    const int pos = len - sr.given + t;
    if (pos < 0) continue;
    const RowRule rr = row_rule(rl, b, pos);
    if (!seen(rl, rr, b, j)) continue;
    for (int h = kh * G; h < kh * G + G; ++h) {
      const int64_t row = sr.r0 + t;
      float a = 0.0f;
      for (int d = 0; d < hd; ++d) a = __builtin_fmaf(static_cast<float>(q[row * q_stride + h * hd + d]), static_cast<float>(k[d]), a);
      const float2 r = mz[row * n_heads + h];
      if (r.y != 0.0f) sum += __builtin_amdgcn_exp2f(simple_score(rl, rl.slopes ? rl.slopes[h] : 0.0f, a, pos, j) - r.x) / r.y;
    }
  }
  *weight_of(kv, page, j, kh) += sum;
}


struct FewPlan {
  int n_blocks, chunk, n_splits, score_len;
  size_t o_bytes, mz_bytes, score_bytes;
};

FewPlan few_plan(const PagedView& kv, const BatchView& bt, int n_heads, int window, bool prefix, int n_cu) {
  FewPlan p{};
  const int group = n_heads / kv.n_kv_heads;
  p.n_blocks = (bt.max_new * group + FEW_ROWS - 1) / FEW_ROWS;
  const int64_t table = static_cast<int64_t>(bt.max_pages) << kv.page_shift;
  int64_t span = std::min<int64_t>(bt.max_len, table);
  p.score_len = static_cast<int>((span + 31) / 32 * 32);
  // rows of a block are at most FEW_ROWS positions apart, lo goes down to a multiple of 32
  if (window > 0 && !prefix) span = std::min<int64_t>(span, static_cast<int64_t>(window) + FEW_ROWS + 32);
  span = std::max<int64_t>(span, 1);
  const int64_t blocks = static_cast<int64_t>(bt.n_seq) * kv.n_kv_heads * p.n_blocks;
  const int64_t chunk = (span * blocks / (FEW_TARGET * n_cu) + FEW_ROUND) / FEW_ROUND * FEW_ROUND;
  p.chunk = static_cast<int>(std::min<int64_t>(std::max<int64_t>(chunk, FEW_MIN_CHUNK), FEW_MAX_CHUNK));
  p.n_splits = static_cast<int>((span + p.chunk - 1) / p.chunk);
  const size_t parts = static_cast<size_t>(bt.n_seq) * bt.max_new * n_heads * p.n_splits;
  if (p.n_splits > 1) p.o_bytes = parts * kv.hd * sizeof(float);
  if (p.n_splits > 1 || kv.weight) p.mz_bytes = (parts * sizeof(float2) + 15) / 16 * 16;
  if (kv.weight) p.score_bytes = static_cast<size_t>(bt.n_seq) * bt.max_new * n_heads * p.score_len * sizeof(float);
  return p;
}

template <typename TC, typename TI, int DP>
hipError_t few(const FewArgs& a, const FewPlan& p, hipStream_t s) {
  const PagedView& kv = a.kv;
  const size_t lds = (static_cast<size_t>(p.chunk >> kv.page_shift) + 2) * sizeof(int64_t);
  hipLaunchKernelGGL((k_attention_few<TC, TI, DP>), dim3(p.n_splits * kv.n_kv_heads * p.n_blocks, a.bt.n_seq), dim3(256), lds, s, a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (p.n_splits > 1) {
    hipLaunchKernelGGL((k_attention_join<TI, DP>), dim3(a.bt.max_new * a.n_heads, a.bt.n_seq), dim3(256), 0, s, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (a.scores) {
    hipLaunchKernelGGL(k_attention_weight, dim3((p.score_len + 255) / 256, kv.n_kv_heads, a.bt.n_seq), dim3(256), 0, s, a);
    return hipGetLastError();
  }
  return hipSuccess;
}

template <typename TC, typename TI>
hipError_t attention(const PagedView& kv, const BatchView& bt, const RuleView& rl, void* out, int64_t out_stride,
                     const void* q, int64_t q_stride, int n_heads, char* scratch, int n_cu, hipStream_t s) {
  const int group = n_heads / kv.n_kv_heads;
  if (static_cast<int64_t>(bt.max_new) * group <= FEW_MOST) {
    const FewPlan p = few_plan(kv, bt, n_heads, rl.window, rl.prefix != nullptr, n_cu);
    FewArgs a{kv, bt, rl, q, out, q_stride, out_stride, n_heads, group, p.n_blocks, p.chunk, p.n_splits,
              reinterpret_cast<float*>(scratch), p.mz_bytes ? reinterpret_cast<float2*>(scratch + p.o_bytes) : nullptr,
              p.score_bytes ? reinterpret_cast<float*>(scratch + p.o_bytes + p.mz_bytes) : nullptr, p.score_len, bt.max_new * group};
    return kv.hd <= 64 ? few<TC, TI, 64>(a, p, s) : kv.hd <= 128 ? few<TC, TI, 128>(a, p, s) : few<TC, TI, 256>(a, p, s);
  }
  float2* mz = kv.weight ? reinterpret_cast<float2*>(scratch) : nullptr;
  hipLaunchKernelGGL((k_paged_attention<TC, TI>), dim3(n_heads, bt.max_new, bt.n_seq), dim3(256), 0, s, kv, bt, rl,
                     static_cast<TI*>(out), out_stride, static_cast<const TI*>(q), q_stride, n_heads, mz);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !mz) return e;
  hipLaunchKernelGGL((k_paged_weight<TC, TI>), dim3((bt.max_len + 255) / 256, kv.n_kv_heads, bt.n_seq), dim3(256), 0, s,
                     kv, bt, rl, static_cast<const TI*>(q), q_stride, n_heads, mz);
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_scratch(const PagedView& kv, const BatchView& bt, const RuleView& rl, int n_heads, int n_cu) {
  if (static_cast<int64_t>(bt.max_new) * (n_heads / kv.n_kv_heads) <= FEW_MOST) {
    const FewPlan p = few_plan(kv, bt, n_heads, rl.window, rl.prefix != nullptr, n_cu);
    return p.o_bytes + p.mz_bytes + p.score_bytes;
  }
  return kv.weight ? static_cast<size_t>(bt.n_rows) * n_heads * sizeof(float2) : 0;
}

hipError_t launch_paged_attention(const PagedView& kv, int kv_type, const BatchView& bt, const RuleView& rl, int io_type,
                                  void* out, int64_t out_stride, const void* q, int64_t q_stride, int n_heads,
                                  void* scratch, int n_cu, hipStream_t s) {
  const bool f32 = io_type == MCPM_TYPE_F32;
  char* sc = static_cast<char*>(scratch);
  if (kv_type == MCPM_TYPE_F32) return attention<float, float>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, sc, n_cu, s);
  if (kv_type == MCPM_TYPE_F16)
    return f32 ? attention<_Float16, float>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, sc, n_cu, s)
               : attention<_Float16, _Float16>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, sc, n_cu, s);
  return f32 ? attention<__bf16, float>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, sc, n_cu, s)
             : attention<__bf16, __bf16>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, sc, n_cu, s);
}

}  // namespace mcpm
