// mcpm_paged_prompt.hip -- attention over the paged cache for many rows: prompts.
//
// A work group takes 128 rows of a sequence and kv head (new tokens x the kv
// head's query heads, token by token, so the heads of a group share every key),
// 32 a wave, and walks the keys in tiles, two LDS buffers in turn: the next
// tile's global loads are in flight while this one is used.  As for single
// tokens the products are formed transposed, S^T = K Q^T and O^T = V^T P^T on the
// 32x32 matrix instructions: a lane's column is one row, its maximum and sum
// need one lane exchange, and the shares are the second product's operand where
// they stand.  For that V goes into LDS turned (by byte permutes on the way) with
// the positions of 16 in the order in which the first product leaves them.
//
// Bound by the issue of matrix and vector instructions, which overlap in part only (a
// share costs an fma, an exp2, a sum and its rounding, as long as the 4 hd flops of its
// two products at hd 64).  4096 new tokens x 16 heads of 128 halves over 16,384
// positions: 584 us, 820 TFLOP/s, the matrix units busy 40 % of the time; a large matrix
// product reaches 1166.  1024 tokens x 32 heads of 64 for 32-bit rows (two terms): 34 us,
// one work group per CU, so prologue, the longest row block's 16 tiles and epilogue in a
// row.  A document mask skips tiles without a document of the rows (three sequences of
// 5003 tokens in documents of 700, 16 heads of 128, capped: 151 us).
#include <climits>

#include "mcpm_paged_score.h"

namespace mcpm {

namespace {

constexpr int PR_ROWS = 128;

// All of `x` in registers here: without it the compiler gives every matrix
// instruction an LDS read of its own to wait for.
template <int N, typename T>
__device__ __forceinline__ void all_here(T (&x)[N]) {
  static_assert(N % 4 == 0);
#pragma unroll
  for (int i = 0; i < N; i += 4) asm volatile("" : "+v"(x[i]), "+v"(x[i + 1]), "+v"(x[i + 2]), "+v"(x[i + 3]));
}

// 16-bit caches: tiles of 64 positions.
template <typename TC, typename TI, int DP>
struct Prompt16 {
  typedef typename Half<TC>::V8 V8;
  static constexpr int NT = Terms<TC, TI>::N;
  static constexpr int KT = 64, KS = DP / 16, NO = DP / 32;
  static constexpr int E = DP >= 128 ? 8 : 4;      // elements of a V load
  static constexpr int NI = DP / (16 * E);         // V loads of a lane and position
  static constexpr int NK = KT * DP / 8 / 256;     // K loads of a lane
  static constexpr int K_STRIDE = DP * 2 + 16, V_STRIDE = KT * 2 + 16;
  static constexpr int BYTES = KT * K_STRIDE + DP * V_STRIDE;
  V8 q[NT][KS];
  f32x16 o[NO];
  float mul;
  u32x4 gk[NK];
  uint32_t gv[NI][4][E / 2];

  // Rows of 32 bits over halves are brought to a top exponent of 8 by a power of
  // two, so that neither term leaves a half's range; products take it back.
  __device__ __forceinline__ void load_q(const TI* row, int hd, float score_mul) {
    typedef TI Row __attribute__((ext_vector_type(8)));
    const int h = (threadIdx.x >> 5) & 1;
    Row x[KS];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bool in = row && 16 * s + 8 * h < hd;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] = static_cast<TI>(0.0f);
      if (in) x[s] = *reinterpret_cast<const Row*>(row + 16 * s + 8 * h);
    }
    mul = score_mul;
    int e = 0;
    if (NT == 2) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(static_cast<float>(x[s][i])));
      top = fmaxf(top, lane_xor32(top));
      if (top > 0.0f && top < __builtin_inff()) {
        e = 9 - __builtin_amdgcn_frexp_expf(top);
        mul = ldexpf(score_mul, -e);
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = NT == 2 ? ldexpf(static_cast<float>(x[s][i]), e) : static_cast<float>(x[s][i]);
      V8 t[NT];
      split_terms<TC, NT>(y, t);
#pragma unroll
      for (int n = 0; n < NT; ++n) q[n][s] = t[n];
    }
#pragma unroll
    for (int j = 0; j < NO; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[j][i] = 0.0f;
  }
  template <class Offset>
  __device__ __forceinline__ void load(const TC* kc, const TC* vc, int p0, int hd, const Offset& offset) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int c = tid + 256 * i;
      gk[i] = *reinterpret_cast<const u32x4*>(kc + offset(p0 + c / (DP / 8)) + min(c % (DP / 8) * 8, hd - 8));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const TC* row = vc + offset(p0 + 4 * (tid >> 4) + r);
#pragma unroll
      for (int it = 0; it < NI; ++it) {
        const TC* p = row + min(E * (16 * it + (tid & 15)), hd - E);
        if constexpr (E == 8) *reinterpret_cast<u32x4*>(gv[it][r]) = *reinterpret_cast<const u32x4*>(p);
        else *reinterpret_cast<u32x2*>(gv[it][r]) = *reinterpret_cast<const u32x2*>(p);
      }
    }
  }
  // The same for a whole tile whose pages hold 16 positions or more: the rows of a
  // wave's load are in one page, so that its address is a scalar base(position) and
  // an offset that a lane keeps.
  uint32_t k_lane, v_lane;
  __device__ __forceinline__ void set_lanes(int hd, uint32_t pos_stride) {
    const int lane = threadIdx.x & 63;
    k_lane = (lane / (DP / 8) * pos_stride + min(lane % (DP / 8) * 8, hd - 8)) * 2;
    v_lane = (4 * (lane >> 4) * pos_stride) * 2;
  }
  template <class Base>
  __device__ __forceinline__ void load_whole(const TC* kc, const TC* vc, int p0, int wave, int hd, int64_t pos_stride, const Base& base) {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const char* p = reinterpret_cast<const char*>(kc + base(p0 + (wave * 64 + 256 * i) / (DP / 8)));
      gk[i] = *reinterpret_cast<const u32x4*>(p + k_lane);
    }
    const TC* v = vc + base(p0 + 16 * wave);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const char* row = reinterpret_cast<const char*>(v + r * pos_stride);
#pragma unroll
      for (int it = 0; it < NI; ++it) {
        const char* p = row + (v_lane + 2 * min(E * (16 * it + static_cast<int>(threadIdx.x & 15)), hd - E));
        if constexpr (E == 8) *reinterpret_cast<u32x4*>(gv[it][r]) = *reinterpret_cast<const u32x4*>(p);
        else *reinterpret_cast<u32x2*>(gv[it][r]) = *reinterpret_cast<const u32x2*>(p);
      }
    }
  }
  __device__ __forceinline__ void store(char* buf) const {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int c = tid + 256 * i;
      *reinterpret_cast<u32x4*>(buf + c / (DP / 8) * K_STRIDE + c % (DP / 8) * 16) = gk[i];
    }
    const int pg = tid >> 4;
    char* v = buf + KT * K_STRIDE + (tid & 15) * V_STRIDE + (pg >> 2) * 32 + (pg & 1) * 16 + (pg >> 1 & 1) * 8;
#pragma unroll
    for (int it = 0; it < NI; ++it)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
        const uint32_t(&r)[4][E / 2] = gv[it];
        *reinterpret_cast<u32x2*>(v + (it * E + j) * 16 * V_STRIDE) =
            u32x2{__builtin_amdgcn_perm(r[1][j / 2], r[0][j / 2], sel), __builtin_amdgcn_perm(r[3][j / 2], r[2][j / 2], sel)};
      }
  }
  // Operands of the products, four 16-byte reads ahead of their use in a ring: of K's
  // KS steps of 16 elements, of V's KS tiles of 32 elements and 16 positions.
  static constexpr int RING = 4;
  V8 k[RING], v[RING];
  static_assert(KS == 2 * NO && KS >= RING);
  __device__ __forceinline__ const char* k_at(const char* buf, int sub) const {
    const int m = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    return buf + (32 * sub + m) * K_STRIDE + h * 16;
  }
  __device__ __forceinline__ const char* v_at(const char* buf, int sub) const {
    const int m = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    return buf + KT * K_STRIDE + m * V_STRIDE + sub * 64 + h * 16;
  }
  __device__ __forceinline__ void read_k(const char* at, int i) { k[i % RING] = *reinterpret_cast<const V8*>(at + i * 32); }
  __device__ __forceinline__ void read_v(const char* at, int i) { v[i % RING] = *reinterpret_cast<const V8*>(at + i % NO * 32 * V_STRIDE + i / NO * 32); }
  __device__ __forceinline__ void begin_k(const char* at) {
#pragma unroll
    for (int i = 0; i < RING; ++i) read_k(at, i);
  }
  __device__ __forceinline__ void score_step(f32x16& s, const char* at, int i) {
#pragma unroll
    for (int n = NT - 1; n >= 0; --n) s = Half<TC>::mma32(k[i % RING], q[n][i], s);
    if (i + RING < KS) read_k(at, i + RING);
  }
  // Scores of the positions whose K begin_k began to read.
  __device__ __forceinline__ void scores(f32x16& s, const char* at) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      score_step(s, at, i);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // A tile's 64 positions in the order in which its two halves overlap best.  Program
  // order is kept (a matrix instruction occupies its unit for 32 cycles, in which the
  // wave issues the vector instructions that follow it): the scores of the second half
  // between the shares of the first, then the first half's outputs between the shares of
  // the second.
  static constexpr int PER = 16 / KS;  // shares to a matrix step
  __device__ __forceinline__ void share(const f32x16& s, float (&p)[16], float scale, float m, float& z, int i) const {
#pragma unroll
    for (int e = i * PER; e < (i + 1) * PER; ++e) {
      p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], scale, -m));
      z += p[e];
    }
  }
  __device__ __forceinline__ void scores_and_shares(f32x16& n, const char* k_base, const f32x16& s, float (&p)[16], float scale, float m, float& z,
                                                    const char* v_base) {
#pragma unroll
    for (int i = 0; i < 16; ++i) n[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      score_step(n, k_base, i);
      if (i >= KS - RING) read_v(v_base, i - (KS - RING));
      share(s, p, scale, m, z, i);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // Outputs of the shares p (V from v_base, its first reads begun); with MORE the
  // shares of s meanwhile, into p2, and the first reads of V at v_after.
  template <bool MORE>
  __device__ __forceinline__ void outputs(const float (&p)[16], const char* v_base, const f32x16& s, float (&p2)[16], float scale, float m, float& z,
                                          const char* v_after) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[8 * ks + i];
      V8 t[NT];
      split_terms<TC, NT>(x, t);
#pragma unroll
      for (int j = 0; j < NO; ++j) {
        const int i = ks * NO + j;
#pragma unroll
        for (int c = NT - 1; c >= 0; --c) o[j] = Half<TC>::mma32(v[i % RING], t[c], o[j]);
        if (i + RING < KS) read_v(v_base, i + RING);
        if constexpr (MORE) {
          if (i >= KS - RING) read_v(v_after, i - (KS - RING));
          share(s, p2, scale, m, z, i);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  // The lane's outputs come in runs of E elements: run c starts at element
  // run_at(c), its element x is o[x / 2][...] as run(c, x) reads it.
  static constexpr int RUN = E, RUNS = DP / (2 * E);
  static __device__ __forceinline__ int run_at(int c) {  // c = (it * 2 + b) * 4 + i
    const int h = (threadIdx.x >> 5) & 1;
    return E * (16 * (c / 8) + 8 * (c / 4 % 2) + 4 * h + c % 4);
  }
  __device__ __forceinline__ float run(int c, int x) const {
    const int t = c / 8 * E + x;  // 16-row group of the turned V
    return o[t / 2][8 * (t % 2) + 4 * (c / 4 % 2) + c % 4];
  }
};
template <typename TC, typename TI, int DP>
struct PromptTile : Prompt16<TC, TI, DP> {};

// 32-bit caches: v_mfma_f32_32x32x2_f32, tiles of 32 positions, K and V as they
// are.  Element c of the 16 bytes that a lane reads goes into instruction c.
template <int DP>
struct PromptTile<float, float, DP> {
  static constexpr int KT = 32, KS = DP / 8, NO = DP / 32;
  static constexpr int W = DP >= 128 ? 4 : 2;     // elements of a V read
  static constexpr int NK = KT * DP / 4 / 256;
  static constexpr int STRIDE = DP * 4 + 16;
  static constexpr int BYTES = 2 * KT * STRIDE;
  f32x4 q[KS];
  f32x16 o[NO];
  float mul;
  u32x4 gk[NK], gv[NK];

  __device__ __forceinline__ void load_q(const float* row, int hd, float score_mul) {
    const int h = (threadIdx.x >> 5) & 1;
    mul = score_mul;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = row && 8 * s < hd ? *reinterpret_cast<const f32x4*>(row + 8 * s + 4 * h) : f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NO; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[j][i] = 0.0f;
  }
  template <class Offset>
  __device__ __forceinline__ void load(const float* kc, const float* vc, int p0, int hd, const Offset& offset) {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int c = threadIdx.x + 256 * i;
      const int64_t at = offset(p0 + c / (DP / 4)) + min(c % (DP / 4) * 4, hd - 4);
      gk[i] = *reinterpret_cast<const u32x4*>(kc + at);
      gv[i] = *reinterpret_cast<const u32x4*>(vc + at);
    }
  }
  uint32_t lane_off;
  __device__ __forceinline__ void set_lanes(int hd, uint32_t pos_stride) {
    const int lane = threadIdx.x & 63;
    lane_off = (lane / (DP / 4) * pos_stride + min(lane % (DP / 4) * 4, hd - 4)) * 4;
  }
  template <class Base>
  __device__ __forceinline__ void load_whole(const float* kc, const float* vc, int p0, int wave, int, int64_t, const Base& base) {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int64_t at = base(p0 + (wave * 64 + 256 * i) / (DP / 4));
      gk[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(kc + at) + lane_off);
      gv[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(vc + at) + lane_off);
    }
  }
  __device__ __forceinline__ void store(char* buf) const {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int c = threadIdx.x + 256 * i;
      char* p = buf + c / (DP / 4) * STRIDE + c % (DP / 4) * 16;
      *reinterpret_cast<u32x4*>(p) = gk[i];
      *reinterpret_cast<u32x4*>(p + KT * STRIDE) = gv[i];
    }
  }
  __device__ __forceinline__ void scores(f32x16& s, const char* buf) const {
    const int m = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    const char* k = buf + m * STRIDE + h * 16;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int i0 = 0; i0 < KS; i0 += 8) {
      f32x4 a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = *reinterpret_cast<const f32x4*>(k + (i0 + i) * 32);
      all_here(a);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) s = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i][c], q[i0 + i][c], s, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void step(const f32x16& s, float scale, float m, float& z, const char* buf) {
    typedef float VecW __attribute__((ext_vector_type(W)));
    const int m32 = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    const char* v = buf + KT * STRIDE + 4 * h * STRIDE + m32 * W * 4;
    float p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale, -m));
      z += p[i];
    }
#pragma unroll
    for (int i0 = 0; i0 < 16; i0 += 4) {
      VecW x[4 * NO / W];
#pragma unroll
      for (int i = 0; i < 4 * NO / W; ++i)
        x[i] = *reinterpret_cast<const VecW*>(v + (2 * i0 + i / (NO / W)) * STRIDE + i % (NO / W) * 32 * W * 4);
      all_here(x);
#pragma unroll
      for (int i = 0; i < 4 * NO / W; ++i)
#pragma unroll
        for (int c = 0; c < W; ++c) {
          const int j = i % (NO / W) * W + c;
          o[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i][c], p[i0 + i / (NO / W)], o[j], 0, 0, 0);
        }
    }
  }
  static constexpr int RUN = W, RUNS = DP / (2 * W);
  static __device__ __forceinline__ int run_at(int c) {  // c = t * 16 + index of the lane's 16 rows
    const int h = (threadIdx.x >> 5) & 1, i = c % 16;
    return W * (32 * (c / 16) + 8 * (i / 4) + 4 * h + i % 4);
  }
  __device__ __forceinline__ float run(int c, int x) const { return o[c / 16 * W + x][c % 16]; }
};

// Waves per SIMD: two where the registers suffice.
template <typename TC, typename TI, int DP>
constexpr int prompt_waves() {
  return DP <= 64 || (DP <= 128 && Terms<TC, TI>::N == 1) ? 2 : 1;
}

template <typename TC, typename TI, int DP>
__global__ void __launch_bounds__(256, (prompt_waves<TC, TI, DP>())) k_attention_prompt(const PagedCall a) {
  typedef PromptTile<TC, TI, DP> Tile;
  constexpr int KT = Tile::KT, SEG = 32 * KT;
  // over halves the shares are taken against 2^-8 of a maximum that may be
  // exceeded 2^7 times before it is raised
  constexpr float LIFT = __is_same(TC, _Float16) ? 8.0f : 0.0f, SLACK = 7.0f;
  __shared__ __attribute__((aligned(16))) char s_tile[2][Tile::BYTES];
  __shared__ __attribute__((aligned(16))) int s_tag[2][KT];
  __shared__ unsigned char s_bad[PR_ROWS];
  __shared__ unsigned s_tiles;
  __shared__ int s_tags[2], s_plain[2];
  extern __shared__ int64_t s_off[];
  const PagedView& kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), n32 = lane & 31, half = lane >> 5;
  // work groups of one sequence and kv head are `pairs` apart, which keeps them on
  // one XCD where pairs divides 8 or the reverse; the rows with the most keys come first
  const int pairs = a.bt.n_seq * kv.n_kv_heads;
  const int pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
  const int b = pair / kv.n_kv_heads, kh = pair % kv.n_kv_heads;
  const int rb = a.n_blocks - 1 - rest % a.n_blocks, split = rest / a.n_blocks;
  const SeqRows sr = seq_rows(a.bt, b);
  const int len = seq_len(a.bt, kv, b);
  if (rb * PR_ROWS >= sr.n * a.group) return;
  const RowBlock fb = row_block(a, b, rb, sr, len);
  const int c0 = fb.keys.lo + split * a.chunk, c1 = min(fb.keys.hi, c0 + a.chunk);
  if (split && c0 >= fb.keys.hi) return;  // the first one answers for rows that see nothing

  const int w0 = rb * PR_ROWS + 32 * wv, r = w0 + n32;
  const bool row_in = r < fb.r_end, wave_in = w0 < fb.r_end;
  const int t = row_in ? r / a.group : 0, head = kh * a.group + (row_in ? r - t * a.group : 0);
  const int64_t row = sr.r0 + t;
  const int pos = fb.pos0 + t;
  const int first = fb.pos0 + w0 / a.group, last = fb.pos0 + (min(w0 + 32, fb.r_end) - 1) / a.group;  // the wave's positions
  const ScoreRule rule = score_rule(a.rl);
  const RowRule rr = row_rule(a.rl, b, row_in ? pos : -1, c1);
  const int prefix = a.rl.prefix ? a.rl.prefix[b] : 0;
  const float slope = a.rl.slopes ? a.rl.slopes[head] * LOG2E : 0.0f;
  const int* docs = a.rl.docs ? a.rl.docs + b * a.rl.docs_stride : nullptr;
  const TC* kc = reinterpret_cast<const TC*>(kv.k) + kh * kv.head_stride;
  const TC* vc = reinterpret_cast<const TC*>(kv.v) + kh * kv.head_stride;

  Tile tile;
  tile.load_q(row_in && pos >= 0 ? static_cast<const TI*>(a.q) + row * a.q_stride + head * kv.hd : nullptr, kv.hd, rule.mul);
  if (tid == 0) {
    s_tags[0] = docs ? INT_MAX : 0;
    s_tags[1] = docs ? -1 : 0;
  }
  __syncthreads();
  if (docs && half == 0 && rr.span) {  // the range of the rows' documents
    atomicMin(&s_tags[0], rr.tag);
    atomicMax(&s_tags[1], rr.tag);
  }

  // a wave's rows in a page, and their offsets in 32 bits
  const bool whole_pages = kv.page_mask >= 15 && kv.pos_stride <= 1 << 24;
  tile.set_lanes(kv.hd, static_cast<uint32_t>(kv.pos_stride));
  const bool all_rows = !__any(row_in && rr.span == 0);  // none that sees nothing

  float m = MAX_START, z = 0.0f;
  for (int seg = c0; seg < c1; seg += SEG) {
    const int seg_end = min(c1, seg + SEG);
    __syncthreads();
    const PagedCall& again = call_again();
    const bool ok = load_page_offsets(again.bt, again.kv, b, seg, seg_end, s_off);
    const int n_tiles = (seg_end - seg + KT - 1) / KT;
    if (tid == 0) s_tiles = docs ? 0u : n_tiles == 32 ? ~0u : (1u << n_tiles) - 1;
    const bool bad_pages = __syncthreads_or(!ok);
    if (docs) {  // tiles that hold a document of these rows
      for (int i = wv; i < n_tiles; i += 4) {
        const int j = seg + i * KT + lane;
        const int d = lane < KT && j < seg_end ? docs[j] : -1;
        if (__any(d >= s_tags[0] && d <= s_tags[1]) && lane == 0) atomicOr(&s_tiles, 1u << i);
      }
      __syncthreads();
    }
    unsigned todo = s_tiles;
    if (!todo) continue;
    const int first_page = seg >> kv.page_shift;
    // element offset of a position's row, of kv head 0; past the segment's end the last one
    auto offset = [&](int j) -> int64_t {
      j = min(j, seg_end - 1);
      return s_off[(j >> kv.page_shift) - first_page] +
             static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(j & kv.page_mask)) * static_cast<uint32_t>(kv.pos_stride));
    };
    // the same of a position that the wave shares, not past the end
    auto base = [&](int j) -> int64_t {
      const uint64_t e = static_cast<uint64_t>(s_off[(j >> kv.page_shift) - first_page]);
      const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(e)), hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(e >> 32));
      return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo) + (j & kv.page_mask) * kv.pos_stride;
    };
    auto load = [&](int p0) {
      if (whole_pages && p0 + KT <= seg_end) tile.load_whole(kc, vc, p0, wv, kv.hd, kv.pos_stride, base);
      else tile.load(kc, vc, p0, kv.hd, offset);
    };
    const bool tagged = docs || bad_pages;
    auto stage_tags = [&](int at, int p0) {
      if (!tagged || wv) return;
      const PagedCall& c = call_again();
      const int tag = lane < KT ? tag_of(c.rl, c.bt, c.kv, b, min(p0 + lane, seg_end - 1), bad_pages) : s_tags[0];
      if (lane < KT) s_tag[at][lane] = tag;
      const bool plain = !__any(tag != s_tags[0]);
      if (lane == 0) s_plain[at] = plain;
    };
    // The rules on the scores of 32 positions, and the running maximum.  Returns what takes
    // the scores to units of log2; `f` gets what the shares so far are multiplied by.
    auto shape = [&](f32x16& s, int p0, int u, int at, float& f) {
      const int pp = p0 + 32 * u;  // the lane: positions pp + 8 (i / 4) + 4 half + i % 4
      // one tag in the tile and in the rows: nothing to tell apart
      const bool tags = tagged && !(s_tags[0] == s_tags[1] && s_plain[at]);
      const bool masked = tags || !all_rows || pp + 31 > first || pp + 32 > seg_end || (a.rl.window > 0 && last - pp >= a.rl.window);
      float scale = tile.mul;
      if (rule.capped || a.rl.slopes || masked || !(rule.mul > 0.0f)) {  // the same for the wave
#pragma unroll
        for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(s[i]));  // nothing of this ahead of the branch
        scale = 1.0f;
        scores_of<16>(rule, s, tile.mul);
        if (a.rl.slopes) {
          const float far = static_cast<float>(pos - (pp + 4 * half));
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(-slope, fabsf(far - static_cast<float>(8 * (i / 4) + i % 4)), s[i]);
        }
        if (masked) {
          const int j0 = pp + 4 * half - rr.lo;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = static_cast<unsigned>(j0 + 8 * (i / 4) + i % 4) < rr.span ? s[i] : -__builtin_inff();
          if (tags) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = s_tag[at][32 * u + 8 * (i / 4) + 4 * half + i % 4] == rr.tag ? s[i] : -__builtin_inff();
          }
        }
      }
      float top = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
      top = __builtin_fmaf(top, scale, -LIFT);
      f = 1.0f;
      if (__any(top > m + SLACK)) {
        top = fmaxf(top, lane_xor32(top));
        const float mn = fmaxf(m, top);
        f = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        z *= f;
#pragma unroll
        for (int j = 0; j < Tile::NO; ++j) tile.o[j] *= f;
      }
      // The shares take s * scale - m with one rounding.  Beyond 2^24 that difference holds
      // the rounding of m, whole units there: the scores are rounded as m was first.
      if (__any(fabsf(m) > 16777216.0f && m > MAX_START)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          asm volatile("" : "+v"(s[i]));
          s[i] *= scale;
        }
        scale = 1.0f;
      }
      return scale;
    };
    int cur = __builtin_ctz(todo), buf = 0;
    todo &= todo - 1;
    load(seg + cur * KT);
    tile.store(s_tile[0]);
    stage_tags(0, seg + cur * KT);
    for (;;) {
      const int next = todo ? __builtin_ctz(todo) : -1;
      todo &= todo - 1;
      __syncthreads();
      if (next >= 0) load(seg + next * KT);
      const int p0 = seg + cur * KT;
      if (wave_in && (p0 <= last || p0 < prefix) && !(a.rl.window > 0 && first - (p0 + KT - 1) >= a.rl.window)) {
        f32x16 s0;
        float p[16], f;
        if constexpr (KT == 64) {
          f32x16 s1;
          float p1[16];
          const char *k0 = tile.k_at(s_tile[buf], 0), *k1 = tile.k_at(s_tile[buf], 1), *v0 = tile.v_at(s_tile[buf], 0), *v1 = tile.v_at(s_tile[buf], 1);
          tile.begin_k(k0);
          tile.scores(s0, k0);
          tile.begin_k(k1);
          float scale = shape(s0, p0, 0, buf, f);
          tile.scores_and_shares(s1, k1, s0, p, scale, m, z, v0);
          scale = shape(s1, p0, 1, buf, f);
          if (__any(f != 1.0f)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] *= f;
          }
          tile.template outputs<true>(p, v0, s1, p1, scale, m, z, v1);
          tile.template outputs<false>(p1, v1, s1, p, scale, m, z, v1);
        } else {
          tile.scores(s0, s_tile[buf]);
          const float scale = shape(s0, p0, 0, buf, f);
          tile.step(s0, scale, m, z, s_tile[buf]);
        }
      }
      if (next < 0) break;
      tile.store(s_tile[buf ^ 1]);
      stage_tags(buf ^ 1, seg + next * KT);
      cur = next;
      buf ^= 1;
    }
  }

  z += lane_xor32(z);
  const PagedCall& c = call_again();
  const bool final = c.n_splits == 1;
  const float inv = z == 0.0f ? 0.0f : 1.0f / z;
  const int64_t at = part_index(c, b, t, head, split);
  bool bad = false;
  if (row_in) {
    bad = !(z < __builtin_inff());
    TI* dst = static_cast<TI*>(c.out) + row * c.out_stride + head * c.kv.hd;
    float* part = c.part_o + at * c.kv.hd;
#pragma unroll
    for (int u = 0; u < Tile::RUNS; ++u) {
      const int d = Tile::run_at(u);
      if (d < c.kv.hd) {
        float x[Tile::RUN];
#pragma unroll
        for (int i = 0; i < Tile::RUN; ++i) {
          x[i] = tile.run(u, i);
          bad = bad || x[i] - x[i] != 0.0f;
        }
#pragma unroll
        for (int i = 0; i < Tile::RUN; ++i) x[i] = final ? x[i] * inv : x[i];
        if (final) {
          typedef TI Out __attribute__((ext_vector_type(Tile::RUN)));
          Out y;
#pragma unroll
          for (int i = 0; i < Tile::RUN; ++i) y[i] = static_cast<TI>(x[i]);
          *reinterpret_cast<Out*>(dst + d) = y;
        } else {
#pragma unroll
          for (int i = 0; i < Tile::RUN; i += 2) *reinterpret_cast<float2*>(part + d + i) = make_float2(x[i], x[i + 1]);
        }
      }
    }
    if (half == 0) {
      if (c.part_mz) c.part_mz[at] = make_float2(m, z);
      if (final && c.row_mz) c.row_mz[row_index(c, b, t, head)] = make_float2(m, z);
    }
  }
  if (!__syncthreads_or(bad)) return;
  // Something infinite or NaN came up: perhaps only a share of 0 times it.
  if (tid < PR_ROWS) s_bad[tid] = 0;
  __syncthreads();
  if (bad) s_bad[r - rb * PR_ROWS] = 1;
  __syncthreads();
  float* lds = reinterpret_cast<float*>(s_tile[0]);
  exact_rows<TC, TI>(b, kh, rb, PR_ROWS, c0, c1, final, s_bad, lds, lds + PAGED_MAX_HD, lds + 2 * PAGED_MAX_HD,
                     [&](const PagedCall& x, int, int tt, int h) { return part_index(x, b, tt, h, split); });
}

template <typename TC, typename TI, int DP>
hipError_t prompt(const PagedCall& a, hipStream_t s) {
  const int64_t grid = static_cast<int64_t>(a.bt.n_seq) * a.kv.n_kv_heads * a.n_blocks * a.n_splits;
  if (grid > INT_MAX) return hipErrorInvalidValue;
  const int seg = 32 * PromptTile<TC, TI, DP>::KT;
  const size_t lds = (static_cast<size_t>(seg >> a.kv.page_shift) + 2) * sizeof(int64_t);
  hipLaunchKernelGGL((k_attention_prompt<TC, TI, DP>), dim3(static_cast<unsigned>(grid)), dim3(256), lds, s, a);
  return hipGetLastError();
}
template <typename TC, typename TI>
hipError_t prompt(const PagedCall& a, hipStream_t s) {
  return a.kv.hd <= 64 ? prompt<TC, TI, 64>(a, s) : a.kv.hd <= 128 ? prompt<TC, TI, 128>(a, s) : prompt<TC, TI, 256>(a, s);
}

}  // namespace

int prompt_block_rows() { return PR_ROWS; }

hipError_t launch_attention_prompt(const PagedCall& a, int kv_type, int io_type, hipStream_t s) {
  const bool f32 = io_type == MCPM_TYPE_F32;
  if (kv_type == MCPM_TYPE_F32) return prompt<float, float>(a, s);
  if (kv_type == MCPM_TYPE_F16) return f32 ? prompt<_Float16, float>(a, s) : prompt<_Float16, _Float16>(a, s);
  return f32 ? prompt<__bf16, float>(a, s) : prompt<__bf16, __bf16>(a, s);
}

}  // namespace mcpm
