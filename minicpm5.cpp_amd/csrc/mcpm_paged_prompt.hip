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
#include <climits>

#include "mcpm_paged_score.h"

namespace mcpm {

namespace {

constexpr int PR_ROWS = 128;

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
    const int h = (threadIdx.x >> 5) & 1;
    int e = 0;
    mul = score_mul;
    if (NT == 2) {
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (row && 16 * s + 8 * h < hd) top = fmaxf(top, fabsf(static_cast<float>(row[16 * s + 8 * h + i])));
      top = fmaxf(top, lane_xor32(top));
      if (top > 0.0f && top < __builtin_inff()) {
        e = 9 - __builtin_amdgcn_frexp_expf(top);
        mul = ldexpf(score_mul, -e);
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = row && 16 * s + 8 * h < hd ? static_cast<float>(row[16 * s + 8 * h + i]) : 0.0f;
      if (NT == 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ldexpf(x[i], e);
      }
      V8 t[NT];
      split_terms<TC, NT>(x, t);
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
  __device__ __forceinline__ f32x16 scores(const char* buf, int sub) const {
    const int m = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    const char* k = buf + (32 * sub + m) * K_STRIDE + h * 16;
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const V8 a = *reinterpret_cast<const V8*>(k + i * 32);
#pragma unroll
      for (int n = NT - 1; n >= 0; --n) s = Half<TC>::mma32(a, q[n][i], s);
    }
    return s;
  }
  __device__ __forceinline__ void add(const char* buf, int sub, const float (&p)[16]) {
    const int m = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    const char* v = buf + KT * K_STRIDE + m * V_STRIDE + sub * 64 + h * 16;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[8 * ks + i];
      V8 t[NT];
      split_terms<TC, NT>(x, t);
#pragma unroll
      for (int j = 0; j < NO; ++j) {
        const V8 a = *reinterpret_cast<const V8*>(v + j * 32 * V_STRIDE + ks * 32);
#pragma unroll
        for (int n = NT - 1; n >= 0; --n) o[j] = Half<TC>::mma32(a, t[n], o[j]);
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
  __device__ __forceinline__ f32x16 scores(const char* buf, int) const {
    const int m = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    const char* k = buf + m * STRIDE + h * 16;
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(k + i * 32);
#pragma unroll
      for (int c = 0; c < 4; ++c) s = __builtin_amdgcn_mfma_f32_32x32x2f32(a[c], q[i][c], s, 0, 0, 0);
    }
    return s;
  }
  __device__ __forceinline__ void add(const char* buf, int, const float (&p)[16]) {
    const int m = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    const char* v = buf + KT * STRIDE + 4 * h * STRIDE + m * W * 4;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const char* row = v + (8 * (i / 4) + i % 4) * STRIDE;
#pragma unroll
      for (int t = 0; t < NO / W; ++t) {
        float x[W];
        if constexpr (W == 4) *reinterpret_cast<f32x4*>(x) = *reinterpret_cast<const f32x4*>(row + t * 32 * W * 4);
        else *reinterpret_cast<u32x2*>(x) = *reinterpret_cast<const u32x2*>(row + t * 32 * W * 4);
#pragma unroll
        for (int c = 0; c < W; ++c) o[t * W + c] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[c], p[i], o[t * W + c], 0, 0, 0);
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

template <typename TC, typename TI, int DP>
__global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) k_attention_prompt(const PagedCall a) {
  typedef PromptTile<TC, TI, DP> Tile;
  constexpr int KT = Tile::KT, SEG = 32 * KT;
  // over halves the shares are taken against 2^-8 of a maximum that may be
  // exceeded 2^7 times before it is raised
  constexpr float LIFT = __is_same(TC, _Float16) ? 8.0f : 0.0f, SLACK = 7.0f;
  __shared__ __attribute__((aligned(16))) char s_tile[2][Tile::BYTES];
  __shared__ __attribute__((aligned(16))) int s_doc[2][KT];
  __shared__ unsigned char s_bad[PR_ROWS];
  __shared__ unsigned s_tiles;
  __shared__ int s_docs[2], s_plain[2];
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
  const RowRule rr = row_rule(a.rl, b, row_in ? pos : -1);
  const int prefix = a.rl.prefix ? a.rl.prefix[b] : 0;
  const float slope = a.rl.slopes ? a.rl.slopes[head] * LOG2E : 0.0f;
  const int* docs = a.rl.docs ? a.rl.docs + b * a.rl.docs_stride : nullptr;
  const TC* kc = reinterpret_cast<const TC*>(kv.k) + kh * kv.head_stride;
  const TC* vc = reinterpret_cast<const TC*>(kv.v) + kh * kv.head_stride;

  Tile tile;
  tile.load_q(row_in && pos >= 0 ? static_cast<const TI*>(a.q) + row * a.q_stride + head * kv.hd : nullptr, kv.hd, rule.mul);
  if (tid == 0) {
    s_docs[0] = INT_MAX;
    s_docs[1] = -1;
  }
  if (tid < PR_ROWS) s_bad[tid] = 0;
  __syncthreads();
  if (docs && half == 0 && rr.pos >= 0) {  // the range of the rows' documents
    atomicMin(&s_docs[0], rr.doc);
    atomicMax(&s_docs[1], rr.doc);
  }

  // a wave's rows in a page, and their offsets in 32 bits
  const bool whole_pages = kv.page_mask >= 15 && kv.pos_stride <= 1 << 24;
  tile.set_lanes(kv.hd, static_cast<uint32_t>(kv.pos_stride));
  const bool all_rows = !__any(row_in && rr.pos < 0);  // none of no document or before the start

  float m = MAX_START, z = 0.0f;
  for (int seg = c0; seg < c1; seg += SEG) {
    const int seg_end = min(c1, seg + SEG);
    __syncthreads();
    const bool ok = load_page_offsets(a.bt, kv, b, seg, seg_end, s_off);
    const int n_tiles = (seg_end - seg + KT - 1) / KT;
    if (tid == 0) s_tiles = docs ? 0u : n_tiles == 32 ? ~0u : (1u << n_tiles) - 1;
    const bool bad_pages = __syncthreads_or(!ok);
    if (docs) {  // tiles that hold a document of these rows
      for (int i = wv; i < n_tiles; i += 4) {
        const int j = seg + i * KT + lane;
        const int d = lane < KT && j < seg_end ? docs[j] : -1;
        if (__any(d >= s_docs[0] && d <= s_docs[1]) && lane == 0) atomicOr(&s_tiles, 1u << i);
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
    int cur = __builtin_ctz(todo), buf = 0;
    todo &= todo - 1;
    load(seg + cur * KT);
    tile.store(s_tile[0]);
    auto stage_docs = [&](int at, int p0) {
      if (!docs || wv) return;
      const int d = lane < KT ? docs[min(p0 + lane, seg_end - 1)] : s_docs[0];
      if (lane < KT) s_doc[at][lane] = d;
      const bool plain = !__any(d != s_docs[0]);
      if (lane == 0) s_plain[at] = plain;
    };
    stage_docs(0, seg + cur * KT);
    for (;;) {
      const int next = todo ? __builtin_ctz(todo) : -1;
      todo &= todo - 1;
      __syncthreads();
      if (next >= 0) load(seg + next * KT);
      const int p0 = seg + cur * KT;
      // one document in the tile and in the rows: nothing to tell apart
      const bool doc_masks = docs && !(s_docs[0] == s_docs[1] && s_plain[buf]);
      if (wave_in && (p0 <= last || p0 < prefix) && !(a.rl.window > 0 && first - (p0 + KT - 1) >= a.rl.window)) {
#pragma unroll
        for (int sub = 0; sub < KT / 32; ++sub) {
          const int pp = p0 + 32 * sub;  // the lane: positions pp + 8 (i / 4) + 4 half + i % 4
          f32x16 s = tile.scores(s_tile[buf], sub);
          const bool masked = doc_masks || !all_rows || bad_pages || pp + 31 > first || pp + 32 > seg_end || (a.rl.window > 0 && last - pp >= a.rl.window);
          const bool shaped = rule.capped || a.rl.slopes || masked || !(rule.mul > 0.0f);  // the same for the wave
          float scale = tile.mul;
          if (shaped) {
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
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int o = 32 * sub + 8 * (i / 4) + 4 * half + i % 4, j = p0 + o;
                bool ok = (j < seg_end) & ((j <= rr.pos) | (j < rr.prefix)) & (rr.pos - j < rr.window);
                if (docs) ok &= s_doc[buf][o] == rr.doc;
                if (bad_pages) ok &= page_of(a.bt, kv, b, min(j, seg_end - 1)) >= 0;
                s[i] = ok ? s[i] : -__builtin_inff();
              }
            }
          }
          float top = s[0];
#pragma unroll
          for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
          top = __builtin_fmaf(top, scale, -LIFT);
          if (__any(top > m + SLACK)) {
            top = fmaxf(top, lane_xor32(top));
            const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            z *= f;
#pragma unroll
            for (int j = 0; j < Tile::NO; ++j) tile.o[j] *= f;
          }
          float p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale, -m));
            z += p[i];
          }
          tile.add(s_tile[buf], sub, p);
        }
      }
      if (next < 0) break;
      tile.store(s_tile[buf ^ 1]);
      stage_docs(buf ^ 1, seg + next * KT);
      cur = next;
      buf ^= 1;
    }
  }

  z += lane_xor32(z);
  const bool final = a.n_splits == 1;
  const float inv = z == 0.0f ? 0.0f : 1.0f / z;
  const int64_t at = part_index(a, b, t, head, split);
  if (row_in) {
    bool bad = !(z < __builtin_inff());
    TI* dst = static_cast<TI*>(a.out) + row * a.out_stride + head * kv.hd;
    float* part = a.part_o + at * kv.hd;
#pragma unroll
    for (int c = 0; c < Tile::RUNS; ++c) {
      const int d = Tile::run_at(c);
      if (d < kv.hd) {
        float x[Tile::RUN];
#pragma unroll
        for (int i = 0; i < Tile::RUN; ++i) {
          x[i] = tile.run(c, i);
          bad = bad || x[i] - x[i] != 0.0f;
        }
#pragma unroll
        for (int i = 0; i < Tile::RUN; ++i)
          if (final) dst[d + i] = static_cast<TI>(x[i] * inv);
          else part[d + i] = x[i];
      }
    }
    if (half == 0 && a.part_mz) a.part_mz[at] = make_float2(m, z);
    if (bad) s_bad[r - rb * PR_ROWS] = 1;
  }
  __syncthreads();
  // Something infinite or NaN came up: perhaps only a share of 0 times it.
  float* lds = reinterpret_cast<float*>(s_tile[0]);
  for (int i = 0; i < PR_ROWS && rb * PR_ROWS + i < fb.r_end; ++i) {
    if (!s_bad[i]) continue;
    const int ri = rb * PR_ROWS + i, ti = ri / a.group, hi = kh * a.group + ri - ti * a.group;
    float2 mz;
    const float o = exact_row<TC, TI>(a, b, kh, sr.r0 + ti, hi, fb.pos0 + ti, c0, c1, lds, lds + PAGED_MAX_HD, lds + 2 * PAGED_MAX_HD, &mz);
    const int64_t ai = part_index(a, b, ti, hi, split);
    if (tid < kv.hd) {
      if (final) static_cast<TI*>(a.out)[(sr.r0 + ti) * a.out_stride + hi * kv.hd + tid] = static_cast<TI>(mz.y == 0.0f ? 0.0f : o / mz.y);
      else a.part_o[ai * kv.hd + tid] = o;
    }
    if (tid == 0 && a.part_mz) a.part_mz[ai] = mz;
  }
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
