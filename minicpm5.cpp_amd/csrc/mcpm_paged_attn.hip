// mcpm_paged_attn.hip -- attention over the paged cache.
//
//   s_j = scale * q.k_j;  cap: c tanh(s/c);  - slope |i - j|;  seen: see mcpm_attn_rules
//   o = sum_j p_j v_j,  p_j = exp(s_j - m) / z over the seen j;  weight_j += p_j
//
// Scores are held in units of log2.
#include <algorithm>
#include <climits>

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
//
// Bound by the bytes of the cache, each read once: two caches of 100,003 positions x 2
// bfloat16 heads of 128, 205 MB, take 43 us (4.8 TB/s, what a large copy reaches) and 7.5
// to join; 48 ragged ones of up to 4099 x 8 heads of 64 halves for 32-bit rows, 251 MB,
// 68 us (3.7 TB/s: work groups of unequal ends, two terms, a capped score and its store)
// and 12.5 to join and weigh; one of 513 x 8 heads of 64, 32 bits, 8.5 us, a chain of
// dependent loads (lengths, pages, rows), and 3.1.

constexpr int FEW_ROWS = 16;
constexpr int FEW_STEP = 32;                // positions of a wave's step
constexpr int FEW_ROUND = 4 * FEW_STEP;     // of a work group's
constexpr int FEW_PAGES = 2048;             // a work group's table of pages in LDS, at most
constexpr int FEW_TARGET = 1, FEW_TARGET_64 = 4;  // work groups per CU that the work is shared among
constexpr int FEW_MOST = 32;                // new tokens x group up to which these kernels run

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
  // A step's rows of K and V.  Two sets, where the registers allow: one is on its way
  // while the other is used.
  struct Rows {
    V8 k[2][KS];
    VRow v[8][VH];
  };
  static constexpr bool AHEAD = DP <= 128;

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
  static __device__ __forceinline__ void load_k(Rows& x, int t, const TC* row, int hd) {
    const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int s = 0; s < KS; ++s) x.k[t][s] = *reinterpret_cast<const V8*>(row + min(32 * s + 8 * g, hd - 8));
  }
  static __device__ __forceinline__ void load_v(Rows& x, int i, const TC* row, int hd) {
    const int m = threadIdx.x & 15;
#pragma unroll
    for (int h = 0; h < VH; ++h) {
      const TC* p = row + min(16 * VW * h + VW * m, hd - VW);
      if constexpr (VW == 8) x.v[i][h].w4 = *reinterpret_cast<const u32x4*>(p);
      else x.v[i][h].w2 = *reinterpret_cast<const u32x2*>(p);
    }
  }
  __device__ __forceinline__ f32x4 scores(const Rows& x, int t) const {
    f32x4 s{0, 0, 0, 0};
#pragma unroll
    for (int n = NT - 1; n >= 0; --n)
#pragma unroll
      for (int i = 0; i < KS; ++i) s = Half<TC>::mma16(x.k[t][i], q[n][i], s);
    return s;
  }
  __device__ __forceinline__ void add(const Rows& x, const float (&p)[8]) {
    V8 t[NT];
    split_terms<TC, NT>(p, t);
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int w = 0; w < VW / 2; ++w) {
        u32x4 lo, hi;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          lo[r] = __builtin_amdgcn_perm(x.v[2 * r + 1][h].w[w], x.v[2 * r][h].w[w], 0x05040100u);
          hi[r] = __builtin_amdgcn_perm(x.v[2 * r + 1][h].w[w], x.v[2 * r][h].w[w], 0x07060302u);
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
  f32x4 q[KS], o[NO];
  float mul;
  struct Rows {
    f32x4 k[2][KS], v[8][VH];
  };
  static constexpr bool AHEAD = DP <= 128;
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
  static __device__ __forceinline__ void load_k(Rows& x, int t, const float* row, int hd) {
    const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int s = 0; s < KS; ++s) x.k[t][s] = *reinterpret_cast<const f32x4*>(row + min(16 * s + 4 * g, hd - 4));
  }
  static __device__ __forceinline__ void load_v(Rows& x, int i, const float* row, int hd) {
    const int m = threadIdx.x & 15;
#pragma unroll
    for (int h = 0; h < VH; ++h) x.v[i][h] = *reinterpret_cast<const f32x4*>(row + min(64 * h + 4 * m, hd - 4));
  }
  __device__ __forceinline__ f32x4 scores(const Rows& x, int t) const {
    f32x4 s{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) s = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[t][i][c], q[i][c], s, 0, 0, 0);
    return s;
  }
  __device__ __forceinline__ void add(const Rows& x, const float (&p)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int h = 0; h < VH; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[4 * h + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[i][h][c], p[i], o[4 * h + c], 0, 0, 0);
  }
  static __device__ __forceinline__ int d_of(int j, int i) {
    const int g = (threadIdx.x >> 4) & 3;
    return 64 * (j / 4) + 4 * (4 * g + i) + j % 4;
  }
};

// A sequence's part of the work: rounds of positions that its rows may see, row blocks.
struct SeqWork {
  KeyRange keys;
  int rounds, blocks;
};
__device__ __forceinline__ SeqWork seq_work(const PagedCall& a, int b) {
  const SeqRows sr = seq_rows(a.bt, b);
  if (!sr.n) return SeqWork{{0, 0}, 0, 0};
  const int len = seq_len(a.bt, a.kv, b), pos0 = len - sr.given;
  const KeyRange k = key_range(a.rl, b, pos0, pos0 + sr.n - 1, len);
  return SeqWork{k, k.hi > k.lo ? (k.hi - k.lo + FEW_ROUND - 1) / FEW_ROUND : 1, (sr.n * a.group + FEW_ROWS - 1) / FEW_ROWS};
}

// Rounds of a work group, at most.
__host__ __device__ inline int few_max_rounds(const PagedView& kv) { return FEW_PAGES / FEW_ROUND << kv.page_shift; }

// Which part of which sequence this work group has.  The host knows a bound of the
// lengths only, and they are ragged: every work group sums up the rounds of all
// sequences and takes its share of them, the same number of rounds (the last of a
// sequence fewer).  Its number is its block index or, with by_xcd (up to 256 sequences),
// counts along the XCDs, so that the heads of a page are read through one L2 and its
// translations (48 ragged caches of 8 heads of 64: 82 us of the call, 87 without; with
// one work group per CU the XCDs' shares are too unequal, 75 us for 65).
struct Share {
  int b, chunk, n_chunks, kh, rb, rounds, first, id;
};
__device__ __forceinline__ bool few_share(const PagedCall& a, Share* s_share, int64_t (*s_wave)[4], Share& out) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, per = a.kv.n_kv_heads, n = a.bt.n_seq;
  SeqWork w = seq_work(a, min(tid, n - 1));
  int64_t sum = 0;
  for (int b = tid; b < n; b += 256) {
    const SeqWork x = b == tid ? w : seq_work(a, b);
    sum += static_cast<int64_t>(x.rounds) * x.blocks * per;
  }
  for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
  if (lane == 0) s_wave[0][wv] = sum;
  if (tid == 0) s_share->b = -1;
  __syncthreads();
  const int64_t total = s_wave[0][0] + s_wave[0][1] + s_wave[0][2] + s_wave[0][3];
  const int rounds = static_cast<int>(min(max((total + a.chunk - 1) / a.chunk, static_cast<int64_t>(1)), static_cast<int64_t>(few_max_rounds(a.kv))));
  int64_t base = 0;
  for (int b0 = 0; b0 < n; b0 += 256) {
    const int b = b0 + tid;
    if (b0 && b < n) w = seq_work(a, b);
    const int chunks = b < n ? (w.rounds + rounds - 1) / rounds : 0;
    const int64_t mine = static_cast<int64_t>(chunks) * w.blocks * per;
    int64_t x = mine;
    for (int s = 1; s < 64; s <<= 1) {
      const int64_t y = __shfl_up(x, s);
      x += lane >= s ? y : 0;
    }
    __syncthreads();
    if (lane == 63) s_wave[1][wv] = x;
    __syncthreads();
    for (int i = 0; i < 4; ++i) x += i < wv ? s_wave[1][i] : 0;
    const int64_t first = base + x - mine;
    int64_t id = blockIdx.x;
    if (a.by_xcd) {
      const int64_t per_xcd = (s_wave[1][0] + s_wave[1][1] + s_wave[1][2] + s_wave[1][3]) / 8;
      if (id < per_xcd * 8) id = id % 8 * per_xcd + id / 8;
    }
    const int64_t i = id - first;
    if (i >= 0 && i < mine) {
      const int k = static_cast<int>(i), pairs = w.blocks * per;
      *s_share = Share{b, k / pairs, chunks, k % per, k % pairs / per, rounds, static_cast<int>(first), static_cast<int>(id)};
    }
    base += s_wave[1][0] + s_wave[1][1] + s_wave[1][2] + s_wave[1][3];
  }
  __syncthreads();
  out = *s_share;
  out.b = __builtin_amdgcn_readfirstlane(out.b);
  out.chunk = __builtin_amdgcn_readfirstlane(out.chunk);
  out.n_chunks = __builtin_amdgcn_readfirstlane(out.n_chunks);
  out.kh = __builtin_amdgcn_readfirstlane(out.kh);
  out.rb = __builtin_amdgcn_readfirstlane(out.rb);
  out.rounds = __builtin_amdgcn_readfirstlane(out.rounds);
  out.first = __builtin_amdgcn_readfirstlane(out.first);
  out.id = __builtin_amdgcn_readfirstlane(out.id);
  return out.b >= 0;
}

template <typename TC, typename TI, int DP>
__global__ void __launch_bounds__(256) k_attention_few(const PagedCall a) {
  __shared__ __attribute__((aligned(16))) float s_o[4][FEW_ROWS][DP + 4];
  __shared__ float s_m[4][FEW_ROWS], s_z[4][FEW_ROWS];
  __shared__ int s_bad;
  extern __shared__ int64_t s_off[];
  const PagedView& kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g = lane >> 4;
  __shared__ Share s_share;
  __shared__ int64_t s_sum[2][4];
  Share sh;
  if (!few_share(a, &s_share, s_sum, sh)) return;
  const int b = sh.b, kh = sh.kh, rb = sh.rb;
  const SeqRows sr = seq_rows(a.bt, b);
  const int len = seq_len(a.bt, kv, b);
  const RowBlock fb = row_block(a, b, rb, sr, len);
  const KeyRange keys = key_range(a.rl, b, fb.pos0, fb.pos0 + sr.n - 1, len);
  const int c0 = keys.lo + sh.chunk * sh.rounds * FEW_ROUND, c1 = min(keys.hi, c0 + sh.rounds * FEW_ROUND);
  const bool final = sh.n_chunks == 1;
  if (sh.id == sh.first && tid == 0 && a.seq_wgs) a.seq_wgs[b] = make_int2(sh.first, sh.n_chunks);

  const int r = rb * FEW_ROWS + n16;
  const bool row_in = r < fb.r_end;
  const int t = row_in ? r / a.group : 0, head = kh * a.group + (row_in ? r - t * a.group : 0);
  const int64_t row = sr.r0 + t;
  const int pos = fb.pos0 + t;
  const ScoreRule rule = score_rule(a.rl);
  const RowRule rr = row_rule(a.rl, b, row_in ? pos : -1, c1);
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

  // over halves the shares are taken against 2^-8 of a maximum that may be
  // exceeded 2^7 times before it is raised: what is down to 2^-22 of it then stays
  // a normal half
  constexpr float LIFT = __is_same(TC, _Float16) ? 8.0f : 0.0f, SLACK = 7.0f;
  float m = MAX_START, z = 0.0f;
  // Rows of one block differ in position by up to 15 tokens: a step that lies
  // before all of them and inside every window needs no masks.
  const bool plain = !a.rl.docs && !bad_pages && fb.first >= 0;
  typedef FewTile<TC, TI, DP> Tile;
  typedef typename Tile::Rows Rows;
  auto load = [&](Rows& x, int p0) {
#pragma unroll
    for (int T = 0; T < 2; ++T) Tile::load_k(x, T, kc + offset(p0 + 16 * T + n16), kv.hd);
#pragma unroll
    for (int i = 0; i < 8; ++i) Tile::load_v(x, i, vc + offset(p0 + 16 * (i >> 2) + 4 * g + (i & 3)), kv.hd);
  };
  auto use = [&](const Rows& rows, int p0) {
    float s[8];
#pragma unroll
    for (int T = 0; T < 2; ++T) {
      const f32x4 x = tile.scores(rows, T);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * T + i] = x[i];
    }
    scores_of<8>(rule, s, tile.mul);
    if (a.rl.slopes) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] -= slope * fabsf(static_cast<float>(pos - (p0 + 16 * (i >> 2) + 4 * g + (i & 3))));
    }
    if (!plain || p0 + FEW_STEP - 1 > fb.first || p0 + FEW_STEP > c1 || (a.rl.window > 0 && fb.last - p0 >= a.rl.window)) {
      const int j0 = p0 + 4 * g - rr.lo;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = static_cast<unsigned>(j0 + 16 * (i >> 2) + (i & 3)) < rr.span ? s[i] : -__builtin_inff();
      if (a.rl.docs || bad_pages) {  // the 32 positions' tags, one a lane
        const int tag = tag_of(a.rl, a.bt, kv, b, min(p0 + (lane & 31), c1 - 1), bad_pages);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int x = __shfl(tag, 16 * (i >> 2) + 4 * g + (i & 3));
          s[i] = x == rr.tag ? s[i] : -__builtin_inff();
        }
      }
    }
    if (sc_row) {
      *reinterpret_cast<f32x4*>(sc_row + p0 + 4 * g) = f32x4{s[0], s[1], s[2], s[3]};
      *reinterpret_cast<f32x4*>(sc_row + p0 + 16 + 4 * g) = f32x4{s[4], s[5], s[6], s[7]};
    }
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7]))) - LIFT;
    if (__any(top > m + SLACK)) {
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
    tile.add(rows, p);
  };
  const int begin = c0 + wv * FEW_STEP;
  if constexpr (Tile::AHEAD) {
    Rows x, y;
    if (begin < c1) load(x, begin);
    for (int p0 = begin; p0 < c1; p0 += 2 * FEW_ROUND) {
      if (p0 + FEW_ROUND < c1) load(y, p0 + FEW_ROUND);
      __builtin_amdgcn_sched_barrier(0);
      use(x, p0);
      if (p0 + FEW_ROUND >= c1) break;
      if (p0 + 2 * FEW_ROUND < c1) load(x, p0 + 2 * FEW_ROUND);
      __builtin_amdgcn_sched_barrier(0);
      use(y, p0 + FEW_ROUND);
    }
  } else {
    Rows x;
    for (int p0 = begin; p0 < c1; p0 += FEW_ROUND) {
      load(x, p0);
      use(x, p0);
    }
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
  const int64_t at = static_cast<int64_t>(sh.id) * FEW_ROWS + rn;
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
  if (in && part == 0) {
    if (a.part_mz) a.part_mz[at] = make_float2(M, Z);
    if (final && a.row_mz) a.row_mz[row_index(a, b, tj, hj)] = make_float2(M, Z);
  }
  if (in && bad) s_bad = 1;
  __syncthreads();
  if (!s_bad) return;
  // Something infinite or NaN came up: perhaps only a share of 0 times it.
  exact_rows<TC, TI>(b, kh, rb, FEW_ROWS, c0, c1, final, nullptr, &s_o[0][0][0], &s_o[2][0][0], &s_m[0][0],
                     [&](const PagedCall&, int i, int, int) { return static_cast<int64_t>(sh.id) * FEW_ROWS + i; });
}

// Where a row's partials are: n of them, `stride` apart.
struct Parts {
  int64_t at, stride;
  int n;
};
template <bool FEW>
__device__ __forceinline__ Parts parts_of(const PagedCall& a, int b, const SeqRows& sr, int t, int head) {
  const int r = t * a.group + head % a.group, rb = r / a.block_rows;
  if constexpr (FEW) {
    const int2 w = a.seq_wgs[b];
    const int blocks = (sr.n * a.group + FEW_ROWS - 1) / FEW_ROWS, per = a.kv.n_kv_heads;
    return Parts{(static_cast<int64_t>(w.x) + rb * per + head / a.group) * FEW_ROWS + r % FEW_ROWS, static_cast<int64_t>(blocks) * per * FEW_ROWS, w.y};
  } else {
    const KeyRange k = row_block(a, b, rb, sr, seq_len(a.bt, a.kv, b)).keys;
    return Parts{part_index(a, b, t, head, 0), 1, k.hi > k.lo ? (k.hi - k.lo + a.chunk - 1) / a.chunk : 1};
  }
}
// (m, z) x joined to mz; returns what the two are multiplied by.
__device__ __forceinline__ float2 join_mz(float2& mz, const float2& x) {
  const float m = fmaxf(mz.x, x.x), f = __builtin_amdgcn_exp2f(mz.x - m), w = __builtin_amdgcn_exp2f(x.x - m);
  mz = make_float2(m, f * mz.y + w * x.y);
  return make_float2(f, w);
}

// The partials of ROWS (new token, head)s into the output, a work group: DP/4 lanes hold
// a row's elements, 256 / (DP/4) / ROWS of them take its partials in turn.
template <bool FEW, typename TI, int DP, int ROWS>
__device__ __forceinline__ void join_rows(const PagedCall& a, int block, int b, char* lds) {
  constexpr int LP = DP / 4, GR = 256 / LP / ROWS;
  f32x4* s_acc = reinterpret_cast<f32x4*>(lds);                       // [ROWS][GR][LP]
  float2* s_mz = reinterpret_cast<float2*>(lds + 256 * sizeof(f32x4));  // [ROWS][GR]
  const int tid = threadIdx.x, hd = a.kv.hd;
  const int e = tid % LP, g = tid / LP % GR, i = tid / LP / GR;
  const SeqRows sr = seq_rows(a.bt, b);
  const int item = block * ROWS + i, t = item / a.n_heads, head = item - t * a.n_heads;
  const bool in = t < sr.n;
  f32x4 acc{0, 0, 0, 0};
  float2 mz = make_float2(MAX_START, 0.0f);
  bool done = !in;
  if (in) {
    const Parts p = parts_of<FEW>(a, b, sr, t, head);
    done = FEW && p.n == 1;  // the work group that had the row stored it
    for (int k = g; k < p.n && !done; k += GR) {
      const int64_t at = p.at + k * p.stride;
      const float2 x = a.part_mz[at];
      if (x.y == 0.0f) continue;
      const f32x4 o = e * 4 < hd ? *reinterpret_cast<const f32x4*>(a.part_o + at * hd + e * 4) : f32x4{0, 0, 0, 0};
      const float2 f = join_mz(mz, x);
      acc = f.x * acc + f.y * o;
    }
  }
  if constexpr (GR > 1) {
    s_acc[(i * GR + g) * LP + e] = acc;
    if (e == 0) s_mz[i * GR + g] = mz;
    __syncthreads();
    if (g) return;
    for (int k = 1; k < GR; ++k) {
      const float2 f = join_mz(mz, s_mz[i * GR + k]);
      acc = f.x * acc + f.y * s_acc[(i * GR + k) * LP + e];
    }
  }
  if (done) return;
  if (e == 0 && a.row_mz) a.row_mz[row_index(a, b, t, head)] = mz;
  if (e * 4 >= hd) return;
  const float inv = mz.y == 0.0f ? 0.0f : 1.0f / mz.y;
  TI* dst = static_cast<TI*>(a.out) + (sr.r0 + t) * a.out_stride + head * hd + e * 4;
#pragma unroll
  for (int k = 0; k < 4; ++k) dst[k] = static_cast<TI>(acc[k] * inv);
}
constexpr int JOIN_LDS = 256 * (sizeof(f32x4) + sizeof(float2));

template <typename TI, int DP, int ROWS>
__global__ void __launch_bounds__(256) k_attention_join(const PagedCall a) {
  __shared__ __attribute__((aligned(16))) char lds[JOIN_LDS];
  join_rows<false, TI, DP, ROWS>(a, blockIdx.x, blockIdx.y, lds);
}

// The weights of 1024 positions of a kv head from the scores: a lane has four, and sums
// the rows in order.  The rows' (m, z) are joined from the partials here too (16 lanes a
// row), so that this runs beside the join.
__device__ __forceinline__ void add_weights(const PagedCall& a, const KeyRange& keys, int kh, int chunk, int b, char* lds) {
  float2* s_mz = reinterpret_cast<float2*>(lds);
  const int tid = threadIdx.x, j = chunk * 1024 + tid * 4;
  const SeqRows sr = seq_rows(a.bt, b);
  const int rows = sr.n * a.group, lane_row = tid / FEW_ROWS, part = tid % FEW_ROWS;
  const float* sc = a.scores + (static_cast<int64_t>(b) * a.kv.n_kv_heads + kh) * a.score_rows * a.score_len + j;
  float* at[4];  // what the sum goes to, asked for ahead of it
  float old[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int page = j + k >= keys.lo && j + k < keys.hi ? page_of(a.bt, a.kv, b, j + k) : -1;
    at[k] = page >= 0 ? weight_of(a.kv, page, j + k, kh) : nullptr;
    old[k] = at[k] ? *at[k] : 0.0f;
  }
  f32x4 sum{0, 0, 0, 0};
  for (int r0 = 0; r0 < rows; r0 += FEW_ROWS) {
    constexpr int AT_ONCE = 4;  // rows whose scores are asked for together
    const f32x4 none = f32x4{0, 0, 0, 0} - __builtin_inff();  // no row: share 0
    f32x4 s[AT_ONCE];
    auto ask = [&](int i0) {
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
        s[i] = j < keys.hi && r0 + i0 + i < rows ? *reinterpret_cast<const f32x4*>(sc + static_cast<int64_t>(r0 + i0 + i) * a.score_len) : none;
    };
    ask(0);
    float2 mz = make_float2(MAX_START, 0.0f);
    if (r0 + lane_row < rows) {
      const int t = (r0 + lane_row) / a.group;
      const Parts p = parts_of<true>(a, b, sr, t, kh * a.group + r0 + lane_row - t * a.group);
      for (int k = part; k < p.n; k += FEW_ROWS) join_mz(mz, a.part_mz[p.at + k * p.stride]);
    }
    for (int x = 1; x < FEW_ROWS; x <<= 1) join_mz(mz, make_float2(__shfl_xor(mz.x, x), __shfl_xor(mz.y, x)));
    __syncthreads();
    if (part == 0) s_mz[lane_row] = make_float2(mz.x, mz.y == 0.0f ? 0.0f : 1.0f / mz.y);
    __syncthreads();
    for (int i0 = 0; i0 < FEW_ROWS && r0 + i0 < rows; i0 += AT_ONCE) {
      if (i0) ask(i0);
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const float2 f = s_mz[i0 + i];
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += j + k >= keys.lo && j + k < keys.hi ? __builtin_amdgcn_exp2f(s[i][k] - f.x) * f.y : 0.0f;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (at[k]) *at[k] = old[k] + sum[k];
}

// After the few-row kernel, in one launch: `join_blocks` work groups a sequence join its
// rows, the others add up the weights.
template <typename TI, int DP, int ROWS>
__global__ void __launch_bounds__(256) k_few_finish(const PagedCall a, int join_blocks, int weight_blocks) {
  __shared__ __attribute__((aligned(16))) char lds[JOIN_LDS];
  const int x = blockIdx.x, b = blockIdx.y, w = x - join_blocks;
  if (w < 0) return join_rows<true, TI, DP, ROWS>(a, x, b, lds);
  const KeyRange keys = seq_work(a, b).keys;
  for (int c = keys.lo / 1024 + w / a.kv.n_kv_heads; c * 1024 < keys.hi; c += weight_blocks) add_weights(a, keys, w % a.kv.n_kv_heads, c, b, lds);
}

// The same where the scores were not kept: they are formed once more.  A work group has
// 64 positions of a kv head, whose keys stay in registers while the rows that may see them
// go by, 16 at a time, the four waves in turn.
constexpr int WEIGHT_KEYS = 64;
template <typename TC, typename TI, int DP>
__device__ __forceinline__ void weights_again(const PagedCall& a, int p0, int kh, int b) {
  typedef FewTile<TC, TI, DP> Tile;
  constexpr int NK = WEIGHT_KEYS / 32;
  __shared__ float s_sum[4][WEIGHT_KEYS];
  const PagedView& kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g = lane >> 4;
  const int len = seq_len(a.bt, kv, b);
  const SeqRows sr = seq_rows(a.bt, b);
  // tokens [t0, t1) may see some of the positions
  const int pos0 = len - sr.given, last = p0 + WEIGHT_KEYS - 1;
  const int t0 = a.rl.prefix && a.rl.prefix[b] > p0 ? 0 : max(p0 - pos0, 0);
  const int t1 = a.rl.window > 0 ? static_cast<int>(min(static_cast<int64_t>(sr.n), max(static_cast<int64_t>(last) - pos0 + a.rl.window, static_cast<int64_t>(0)))) : sr.n;
  if (t0 >= t1) return;

  typename Tile::Rows keys[NK];
  int tag[NK][8];
#pragma unroll
  for (int n = 0; n < NK; ++n) {
#pragma unroll
    for (int T = 0; T < 2; ++T) {
      const int j = min(p0 + 32 * n + 16 * T + n16, len - 1);
      Tile::load_k(keys[n], T, reinterpret_cast<const TC*>(kv.k) + elem_of(kv, max(page_of(a.bt, kv, b, j), 0), j, kh), kv.hd);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) tag[n][i] = tag_of(a.rl, a.bt, kv, b, min(p0 + 32 * n + 16 * (i >> 2) + 4 * g + (i & 3), len - 1), true);
  }
  const ScoreRule rule = score_rule(a.rl);
  float sum[NK][8] = {};
  for (int r0 = t0 * a.group + 16 * wv; r0 < t1 * a.group; r0 += 64) {
    const int r = r0 + n16;
    const bool in = r < t1 * a.group;
    const int t = in ? r / a.group : t0, head = kh * a.group + (in ? r - t * a.group : 0), pos = pos0 + t;
    const float2 mz = a.row_mz[row_index(a, b, t, head)];
    const float inv = in && mz.y != 0.0f ? 1.0f / mz.y : 0.0f;
    const RowRule rr = row_rule(a.rl, b, in ? pos : -1, len);
    const float slope = a.rl.slopes ? a.rl.slopes[head] * LOG2E : 0.0f;
    const int j0 = p0 + 4 * g;
    Tile tile;
    tile.load_q(static_cast<const TI*>(a.q) + (sr.r0 + t) * a.q_stride + head * kv.hd, kv.hd, rule.mul);
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      float s[8];
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        const f32x4 x = tile.scores(keys[n], T);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * T + i] = x[i];
      }
      scores_of<8>(rule, s, tile.mul);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + 32 * n + 16 * (i >> 2) + (i & 3);
        const float x = s[i] - slope * fabsf(static_cast<float>(pos - j));
        sum[n][i] += in_span(rr, j) && tag[n][i] == rr.tag ? __builtin_amdgcn_exp2f(x - mz.x) * inv : 0.0f;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NK; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = sum[n][i];
      for (int k = 1; k < 16; k <<= 1) x += __shfl_xor(x, k);
      if (n16 == 0) s_sum[wv][32 * n + 16 * (i >> 2) + 4 * g + (i & 3)] = x;
    }
  __syncthreads();
  if (tid < WEIGHT_KEYS && p0 + tid < len) {
    const int page = page_of(a.bt, kv, b, p0 + tid);
    if (page >= 0) *weight_of(kv, page, p0 + tid, kh) += s_sum[0][tid] + s_sum[1][tid] + s_sum[2][tid] + s_sum[3][tid];
  }
  __syncthreads();
}
template <typename TC, typename TI, int DP>
__global__ void __launch_bounds__(256) k_prompt_weight(const PagedCall a) {
  const int len = seq_len(a.bt, a.kv, blockIdx.z);
  for (int p0 = blockIdx.x * WEIGHT_KEYS; p0 < len; p0 += gridDim.x * WEIGHT_KEYS) weights_again<TC, TI, DP>(call_again(), p0, blockIdx.y, blockIdx.z);
}

// How a call is cut into work groups.  Up to FEW_MOST rows of a sequence and kv
// head take the 16-row kernel, more the prompt kernel.
struct Plan {
  bool few, by_xcd;
  int block_rows, n_blocks, chunk, n_splits, grid, lds_pages, row_parts, score_len;
  size_t o_bytes, mz_bytes, row_bytes, seq_bytes, score_bytes;
  size_t bytes() const { return o_bytes + mz_bytes + row_bytes + seq_bytes + score_bytes; }
};
size_t round16(size_t n) { return (n + 15) / 16 * 16; }
constexpr size_t MOST_SCORES = size_t{1} << 30;  // bytes of kept scores, past which they are formed again

// Work groups per CU that a prompt's length is split for, and the shortest chunk.  A
// split pays for its join where a tile of keys is dear: on the 32-bit matrix
// instructions, 1/8 of the rate, anywhere (heads of 256, 200 tokens: 82 us whole, 48 in
// chunks of 64), there with four work groups per CU, which even out the causal triangle
// (heads of 128, 2400 tokens: 381 us with one, 240 with four; under a window or with
// documents, which leave no triangle, one: 164 us, 242 with four); with heads of 256 or 32-bit rows over a
// 16-bit cache's heads of 128 in chunks of 128 (1000 tokens, 8 heads of 256: 124 us
// whole, 82 split); not elsewhere (300 tokens, heads of 64: 12 us whole, 15 split), nor
// over 16 bits where documents leave most of a chunk unseen (260 tokens in documents of
// 30, heads of 256: 38 us whole, 44 split).
struct PromptSplit {
  int per_cu, least;
};
PromptSplit prompt_split(int kv_type, int io_type, int hd, const RuleView& rl) {
  if (kv_type == MCPM_TYPE_F32) return {rl.docs || (rl.window > 0 && !rl.prefix) ? 1 : 4, 64};
  if (rl.docs) return {1, 512};
  return {1, hd > 128 || (hd > 64 && io_type == MCPM_TYPE_F32) ? 128 : 512};
}

Plan plan_of(const PagedView& kv, int kv_type, const BatchView& bt, const RuleView& rl, int io_type, int n_heads, int n_cu) {
  Plan p{};
  const int group = n_heads / kv.n_kv_heads;
  const int64_t rows = static_cast<int64_t>(bt.max_new) * group;
  p.few = rows <= FEW_MOST;
  p.block_rows = p.few ? FEW_ROWS : prompt_block_rows();
  p.n_blocks = static_cast<int>((rows + p.block_rows - 1) / p.block_rows);
  const int64_t table = static_cast<int64_t>(bt.max_pages) << kv.page_shift;
  int64_t span = std::min<int64_t>(bt.max_len, table);
  p.score_len = static_cast<int>((span + 63) / 64 * 64);
  // rows of a block are at most block_rows positions apart, lo goes down to a multiple of 64
  if (rl.window > 0 && !rl.prefix) span = std::min<int64_t>(span, static_cast<int64_t>(rl.window) + std::max(p.block_rows, FEW_MOST) + 64);
  span = std::max<int64_t>(span, 1);
  const int64_t blocks = static_cast<int64_t>(bt.n_seq) * kv.n_kv_heads * p.n_blocks;
  size_t parts;
  if (p.few) {
    const int64_t rounds = (span + FEW_ROUND - 1) / FEW_ROUND;
    // One work group per CU keeps its memory busy, and more of them start later (two
    // caches of 100,003, heads of 128: 50 us, 61 with two).  Heads of up to 64 leave room
    // for more at once, which evens out many ragged sequences of costly rules (48 with
    // weights and a cap: 82 us instead of 97; a single one of 40,000 loses, 33 for 25).
    const bool many = kv.hd <= 64 && blocks >= n_cu;
    const int per_cu = many ? FEW_TARGET_64 : FEW_TARGET;
    p.by_xcd = many && bt.n_seq <= 256;
    p.chunk = per_cu * n_cu;
    // few_share gives a block a work group more than its share, at most, and none more than max_rounds
    const int max_rounds = few_max_rounds(kv);
    const int64_t most = std::max<int64_t>(p.chunk, blocks * ((rounds + max_rounds - 1) / max_rounds)) + blocks;
    p.lds_pages = static_cast<int>(std::min<int64_t>(FEW_PAGES, span >> kv.page_shift) + 2);
    const int64_t grid = std::min(most, blocks * rounds);
    p.grid = grid > INT_MAX ? -1 : static_cast<int>(grid);
    p.n_splits = rounds > 1 ? 2 : 1;
    p.row_parts = static_cast<int>(std::min<int64_t>((p.chunk + blocks - 1) / blocks, rounds));  // about
    parts = static_cast<size_t>(grid) * FEW_ROWS;
    p.seq_bytes = p.n_splits > 1 || kv.weight ? round16(bt.n_seq * sizeof(int2)) : 0;
  } else {
    const PromptSplit split = prompt_split(kv_type, io_type, kv.hd, rl);
    const int64_t want = std::max<int64_t>(1, static_cast<int64_t>(split.per_cu) * n_cu / blocks);
    p.chunk = static_cast<int>((std::max<int64_t>((span + want - 1) / want, split.least) + 63) / 64 * 64);
    p.row_parts = p.n_splits = static_cast<int>((span + p.chunk - 1) / p.chunk);
    parts = static_cast<size_t>(bt.n_seq) * bt.max_new * n_heads * p.n_splits;
  }
  const size_t all_rows = static_cast<size_t>(bt.n_seq) * bt.max_new * n_heads;
  if (p.n_splits > 1) p.o_bytes = parts * kv.hd * sizeof(float);
  if (p.n_splits > 1 || (kv.weight && p.few)) p.mz_bytes = round16(parts * sizeof(float2));
  if (kv.weight) {
    p.score_bytes = p.few ? all_rows * p.score_len * sizeof(float) : 0;
    if (p.score_bytes > MOST_SCORES) p.score_bytes = 0;
    if (!p.score_bytes) p.row_bytes = round16(all_rows * sizeof(float2));
  }
  return p;
}

template <typename TC, typename TI, int DP>
hipError_t few(const PagedCall& a, const Plan& p, hipStream_t s) {
  hipLaunchKernelGGL((k_attention_few<TC, TI, DP>), dim3(p.grid), dim3(256), p.lds_pages * sizeof(int64_t), s, a);
  return hipGetLastError();
}
template <typename TC, typename TI>
hipError_t few(const PagedCall& a, const Plan& p, hipStream_t s) {
  return a.kv.hd <= 64 ? few<TC, TI, 64>(a, p, s) : a.kv.hd <= 128 ? few<TC, TI, 128>(a, p, s) : few<TC, TI, 256>(a, p, s);
}
hipError_t launch_attention_few(const PagedCall& a, const Plan& p, int kv_type, int io_type, hipStream_t s) {
  if (p.grid < 0) return hipErrorInvalidValue;
  const bool f32 = io_type == MCPM_TYPE_F32;
  if (kv_type == MCPM_TYPE_F32) return few<float, float>(a, p, s);
  if (kv_type == MCPM_TYPE_F16) return f32 ? few<_Float16, float>(a, p, s) : few<_Float16, _Float16>(a, p, s);
  return f32 ? few<__bf16, float>(a, p, s) : few<__bf16, __bf16>(a, p, s);
}

// Work groups for each (sequence, kv head) of a weights' sum over `most` slices: per_cu
// of them per CU in all, so that a bound far above the lengths costs no idle ones.
int slices_of(int most, int per_cu, const PagedCall& a, int n_cu) {
  const int64_t pairs = static_cast<int64_t>(a.bt.n_seq) * a.kv.n_kv_heads;
  return static_cast<int>(std::min<int64_t>(most, (static_cast<int64_t>(per_cu) * n_cu + pairs - 1) / pairs));
}

// What follows the main kernel: the join where rows are in parts, the weights' sum
// where the scores were kept.
template <typename TI, int DP>
hipError_t finish(const PagedCall& a, const Plan& p, int n_cu, hipStream_t s) {
  constexpr int LP = DP / 4, MOST = 256 / LP;
  const int items = a.bt.max_new * a.n_heads, groups = a.n_splits > 1 ? (items + MOST - 1) / MOST : 0;
  // rows side by side in a work group where they have few partials or fill the CUs so (48
  // caches in 3 each save 3 us of the call), a row's partials where they are many
  // (two of 100,003 in 64 each: 51 us, 80 side by side)
  const bool side = p.row_parts <= 4 || static_cast<int64_t>(items) * a.bt.n_seq >= static_cast<int64_t>(MOST) * n_cu;
  const int joins = a.n_splits == 1 ? 0 : side ? groups : items;
  if (!p.few) {
    if (side) hipLaunchKernelGGL((k_attention_join<TI, DP, MOST>), dim3(joins, a.bt.n_seq), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_attention_join<TI, DP, 1>), dim3(joins, a.bt.n_seq), dim3(256), 0, s, a);
  } else {
    const int weights = a.scores ? slices_of((a.score_len + 1023) / 1024, 8, a, n_cu) : 0;
    const dim3 grid(joins + weights * a.kv.n_kv_heads, a.bt.n_seq);
    if (side) hipLaunchKernelGGL((k_few_finish<TI, DP, MOST>), grid, dim3(256), 0, s, a, joins, weights);
    else hipLaunchKernelGGL((k_few_finish<TI, DP, 1>), grid, dim3(256), 0, s, a, joins, weights);
  }
  return hipGetLastError();
}
template <typename TI>
hipError_t finish(const PagedCall& a, const Plan& p, int n_cu, hipStream_t s) {
  return a.kv.hd <= 64 ? finish<TI, 64>(a, p, n_cu, s) : a.kv.hd <= 128 ? finish<TI, 128>(a, p, n_cu, s) : finish<TI, 256>(a, p, n_cu, s);
}

template <typename TC, typename TI, int DP>
hipError_t prompt_weight(const PagedCall& a, int n_cu, hipStream_t s) {
  const dim3 grid(slices_of((a.score_len + WEIGHT_KEYS - 1) / WEIGHT_KEYS, 32, a, n_cu), a.kv.n_kv_heads, a.bt.n_seq);
  hipLaunchKernelGGL((k_prompt_weight<TC, TI, DP>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}
template <typename TC, typename TI>
hipError_t prompt_weight(const PagedCall& a, int n_cu, hipStream_t s) {
  return a.kv.hd <= 64 ? prompt_weight<TC, TI, 64>(a, n_cu, s) : a.kv.hd <= 128 ? prompt_weight<TC, TI, 128>(a, n_cu, s) : prompt_weight<TC, TI, 256>(a, n_cu, s);
}

}  // namespace

size_t paged_attention_scratch(const PagedView& kv, int kv_type, const BatchView& bt, const RuleView& rl, int io_type, int n_heads, int n_cu) {
  return plan_of(kv, kv_type, bt, rl, io_type, n_heads, n_cu).bytes();
}

hipError_t launch_paged_attention(const PagedView& kv, int kv_type, const BatchView& bt, const RuleView& rl, int io_type,
                                  void* out, int64_t out_stride, const void* q, int64_t q_stride, int n_heads,
                                  void* scratch, int n_cu, hipStream_t s) {
  const Plan p = plan_of(kv, kv_type, bt, rl, io_type, n_heads, n_cu);
  const int group = n_heads / kv.n_kv_heads;
  char* sc = static_cast<char*>(scratch);
  auto take = [&](size_t bytes) {
    char* at = bytes ? sc : nullptr;
    sc += bytes;
    return at;
  };
  PagedCall a{kv, bt, rl, q, out, q_stride, out_stride, n_heads, group, p.block_rows, p.n_blocks, p.chunk, p.n_splits, p.by_xcd};
  a.part_o = reinterpret_cast<float*>(take(p.o_bytes));
  a.part_mz = reinterpret_cast<float2*>(take(p.mz_bytes));
  a.row_mz = reinterpret_cast<float2*>(take(p.row_bytes));
  a.seq_wgs = reinterpret_cast<int2*>(take(p.seq_bytes));
  a.scores = reinterpret_cast<float*>(take(p.score_bytes));
  a.score_len = p.score_len;
  a.score_rows = bt.max_new * group;
  hipError_t e = p.few ? launch_attention_few(a, p, kv_type, io_type, s) : launch_attention_prompt(a, kv_type, io_type, s);
  if (e != hipSuccess) return e;
  if (p.n_splits > 1 || a.scores) {
    e = io_type == MCPM_TYPE_F32 ? finish<float>(a, p, n_cu, s) : io_type == MCPM_TYPE_F16 ? finish<_Float16>(a, p, n_cu, s) : finish<__bf16>(a, p, n_cu, s);
    if (e != hipSuccess) return e;
  }
  if (!kv.weight || a.scores || !p.score_len) return hipSuccess;
  const bool f32 = io_type == MCPM_TYPE_F32;
  if (kv_type == MCPM_TYPE_F32) return prompt_weight<float, float>(a, n_cu, s);
  if (kv_type == MCPM_TYPE_F16) return f32 ? prompt_weight<_Float16, float>(a, n_cu, s) : prompt_weight<_Float16, _Float16>(a, n_cu, s);
  return f32 ? prompt_weight<__bf16, float>(a, n_cu, s) : prompt_weight<__bf16, __bf16>(a, n_cu, s);
}

}  // namespace mcpm
