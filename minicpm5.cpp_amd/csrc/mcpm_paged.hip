// mcpm_paged.hip -- writing side of the paged cache: the append of new tokens
// (with the rotation of k and q) and the eviction by accumulated weight.
#include <climits>
#include <cmath>

#include "mcpm_device.h"
#include "mcpm_paged.h"

namespace mcpm {

namespace {

// ------------------------------------------------------------- append ------

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  return static_cast<float>(v);
}

// 8 consecutive elements.
template <typename T>
struct alignas(sizeof(T) * 8 < 16 ? sizeof(T) * 8 : 16) Vec8 {
  T v[8];
};

// One work group per row (and slice of its heads).  A row's angles are the same
// for all heads: hd/2 lanes form them once in 64 bits, reduced to a turn before
// the sine, and leave (cos, sin) in LDS.  Then a lane turns and moves 8 elements.
// Bound by the copy for prompts (8800 bfloat16 rows of 16 + 2 + 2 heads of 128, 90 MB:
// 19.0 us, 4.8 TB/s, what a large copy reaches), by the launch for single tokens (64
// rows: 4.2 us).
template <typename TC, typename TI>
__global__ void __launch_bounds__(256) k_paged_append(PagedView kv, BatchView bt, const TI* __restrict__ k,
                                                      const TI* __restrict__ v, int64_t kv_stride, TI* __restrict__ q,
                                                      int64_t q_stride, int n_heads, double log2_base, int rotate) {
  __shared__ float2 cs[PAGED_MAX_HD / 2];
  const int row = blockIdx.x, tid = threadIdx.x, hd = kv.hd;
  // the sequence whose rows hold this one
  int b = row;
  if (bt.starts) {
    int lo = 0, hi = bt.n_seq;  // starts[lo] <= row < starts[hi]
    if (row < bt.starts[0] || row >= bt.starts[bt.n_seq]) return;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (bt.starts[mid] <= row) lo = mid;
      else hi = mid;
    }
    b = lo;
  }
  if (b >= bt.n_seq) return;
  const SeqRows sr = seq_rows(bt, b);
  const int t = row - sr.r0;
  if (t < 0 || t >= sr.n) return;
  const int pos = seq_len(bt, kv, b) - sr.given + t;
  if (pos < 0) return;
  if (rotate) {
    if (tid < hd / 2) {
      const double theta = exp2(-log2_base * (2.0 * tid / hd));
      const double turns = pos * theta * 0.15915494309189533577;
      double sn, c;
      sincospi(2.0 * (turns - rint(turns)), &sn, &c);
      cs[tid] = make_float2(static_cast<float>(c), static_cast<float>(sn));
    }
    __syncthreads();
  }
  const int page = page_of(bt, kv, b, pos);
  const int per = hd / 8, nk = kv.n_kv_heads * per, nq = q && rotate ? n_heads * per : 0;
  TC* kc = reinterpret_cast<TC*>(kv.k);
  TC* vc = reinterpret_cast<TC*>(kv.v);
  for (int c = blockIdx.y * 256 + tid; c < 2 * nk + nq; c += 256 * gridDim.y) {
    const bool is_v = c >= nk && c < 2 * nk, is_q = c >= 2 * nk;
    const int cc = is_q ? c - 2 * nk : is_v ? c - nk : c;
    const int h = cc / per, d = (cc - h * per) * 8;
    if (!is_q && page < 0) continue;
    TI* src = is_q ? q + row * q_stride + h * hd + d
                   : const_cast<TI*>((is_v ? v : k) + row * kv_stride + h * hd + d);
    const Vec8<TI> in = *reinterpret_cast<const Vec8<TI>*>(src);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f(in.v[i]);
    if (rotate && !is_v) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float2 a = cs[(d + i) / 2];
        const float x0 = x[i], x1 = x[i + 1];
        x[i] = x0 * a.x - x1 * a.y;
        x[i + 1] = x0 * a.y + x1 * a.x;
      }
    }
    if (is_q) {
      Vec8<TI> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[i] = static_cast<TI>(x[i]);
      *reinterpret_cast<Vec8<TI>*>(src) = o;
    } else {
      Vec8<TC> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[i] = static_cast<TC>(x[i]);
      *reinterpret_cast<Vec8<TC>*>((is_v ? vc : kc) + elem_of(kv, page, pos, h) + d) = o;
      if (kv.weight && !is_v && d == 0) *weight_of(kv, page, pos, h) = 0.0f;
    }
  }
}

// ------------------------------------------------------------- evict -------

// A float's order as unsigned: larger weight, larger key; NaN below all.
__device__ __forceinline__ unsigned weight_key(float w) {
  if (w != w) return 0u;
  const unsigned u = __float_as_uint(w == 0.0f ? 0.0f : w);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr int EV_T = 1024;

// For each of N counts: the sum over the lanes before this one in the work group;
// `all` gets the sums over every lane.
template <int N, int WAVES>
__device__ __forceinline__ void block_prefix(int (&v)[N], int (*s_wave)[WAVES], int (&all)[N]) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int x[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    x[n] = v[n];
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int y = __shfl_up(x[n], s);
      x[n] += lane >= s ? y : 0;
    }
  }
  __syncthreads();
  if (lane == 63)
#pragma unroll
    for (int n = 0; n < N; ++n) s_wave[n][wv] = x[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int before = 0;
    all[n] = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const int c = s_wave[n][w];
      before += w < wv ? c : 0;
      all[n] += c;
    }
    v[n] = before + x[n] - v[n];
  }
}

// The keys of V consecutive positions from j, a multiple of V, on; 0 outside
// [first, end).  Inside one page wherever pages hold that many: 16-byte loads.
template <int V>
__device__ __forceinline__ void load_keys(const PagedView& kv, const BatchView& bt, int b, int h, int j, int end, unsigned (&key)[V]) {
  if (kv.page_mask >= V - 1) {
    const int page = j < end ? page_of(bt, kv, b, j) : -1;
    f32x4 w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = page >= 0 ? *reinterpret_cast<const f32x4*>(weight_of(kv, page, j, h) + 4 * i) : f32x4{NAN, NAN, NAN, NAN};
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = weight_key(w[i / 4][i % 4]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int page = j + i < end ? page_of(bt, kv, b, j + i) : -1;
      key[i] = page >= 0 ? weight_key(*weight_of(kv, page, j + i, h)) : 0u;
    }
  }
}

// What is kept whatever it weighs, and the end of the list.  Returns whether there is
// anything to choose.
__device__ __forceinline__ bool kept_ends(int len, int budget, int first, int recent, int lane, int lanes, int* out) {
  for (int i = min(len, budget) + lane; i < budget; i += lanes) out[i] = -1;
  if (len <= budget) {
    for (int i = lane; i < len; i += lanes) out[i] = i;
    return false;
  }
  for (int i = lane; i < first; i += lanes) out[i] = i;
  for (int i = lane; i < recent; i += lanes) out[budget - recent + i] = len - recent + i;
  return budget - first - recent > 0;
}

// The bin, from the top, in which the running count reaches `need`: BINS counts
// in LDS, PER a lane (lane t has the ones that end at BINS - 1 - PER t).
struct Edge {
  int bin, need, count;  // the bin, how many of its values are needed, how many it has
};
template <int PER, int WAVES>
__device__ __forceinline__ void find_edge(const int* hist, int bins, int need, int (*s_wave)[WAVES], Edge* s_edge) {
  const int top = bins - 1 - PER * static_cast<int>(threadIdx.x);
  int c[PER], sum[1] = {0}, total[1];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = hist[top - i];
    sum[0] += c[i];
  }
  const int mine = sum[0];
  block_prefix(sum, s_wave, total);
  int above = sum[0];
  if (above < need && above + mine >= need) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (above < need && above + c[i] >= need) *s_edge = Edge{top - i, need - above, c[i]};
      above += c[i];
    }
  }
  __syncthreads();
}

// Up to 16 x 1024 candidates: one work group per (sequence, kv head).  A lane has
// V consecutive positions, whose keys stay in registers.  The key of the smallest weight
// kept comes from histograms of 11, 11 and 10 bits: the first one has the weight's
// exponent and two bits of its fraction, so that lanes seldom meet in a bin, the
// others count only what is left.  Kept then are the larger keys and, of those
// equal to it, the first ones.  Bound by its chain of barriers: three passes of
// clear, count, prefix (8 caches of 4096 x 8 heads: 7.5 us, and 7.5 for the copy).
constexpr int EV_BINS = 2048;

template <int V>
__global__ void __launch_bounds__(EV_T) k_evict_select(PagedView kv, BatchView bt, int budget, int first, int recent,
                                                       int* __restrict__ kept, int* __restrict__ dst_lens) {
  __shared__ int hist[EV_BINS];
  __shared__ int s_wave[1][EV_T / 64];
  __shared__ Edge s_edge;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int len = seq_len(bt, kv, b);
  int* out = kept + (static_cast<int64_t>(b) * kv.n_kv_heads + h) * budget;
  if (h == 0 && tid == 0) dst_lens[b] = min(len, budget);
  if (!kept_ends(len, budget, first, recent, tid, EV_T, out)) return;
  const int begin = first & ~(V - 1), end = len - recent;  // candidates are [first, end)
  const int j0 = begin + tid * V;
  unsigned key[V];
  load_keys<V>(kv, bt, b, h, j0, end, key);
  // bit i: position i of the lane's is a candidate (bits, for V conditions held through the
  // passes would fill the scalar registers)
  unsigned cand = ((1u << min(max(end - j0, 0), V)) - 1) & ~((1u << min(max(first - j0, 0), V)) - 1);
  auto candidate = [&](int i) { return (cand >> i & 1) != 0; };
  auto held = [&] { asm volatile("" : "+v"(cand)); };
  unsigned edge = 0;
  int need = budget - first - recent;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : EV_BINS;
    const unsigned mask = pass == 0 ? 0u : pass == 1 ? ~0u << 21 : ~0u << 10;
    for (int i = tid; i < EV_BINS; i += EV_T) hist[i] = 0;
    __syncthreads();
    held();
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (candidate(i) && (key[i] & mask) == edge) atomicAdd(&hist[(key[i] >> shift) & (bins - 1)], 1);
    __syncthreads();
    find_edge<EV_BINS / EV_T>(hist, EV_BINS, need, s_wave, &s_edge);
    edge |= static_cast<unsigned>(s_edge.bin) << shift;
    need = s_edge.need;
  }
  held();
  unsigned keep = 0;  // bit i: position i of the lane's is kept
  int n[1] = {0}, all[1];
  if (s_edge.count != need) {  // the first `need` of the equal ones
#pragma unroll
    for (int i = 0; i < V; ++i) n[0] += candidate(i) && key[i] == edge;
    block_prefix(n, s_wave, all);
  } else {
    need = INT_MAX;
  }
  int rank = n[0];
  held();
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (candidate(i) && (key[i] > edge || (key[i] == edge && rank++ < need))) keep |= 1u << i;
  n[0] = __popc(keep);
  block_prefix(n, s_wave, all);
  int o = first + n[0];
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (keep >> i & 1) out[o++] = j0 + i;
}

// More candidates: the same over slices of SL_T x SL_V positions, a work group
// each, in three launches, for one CU has neither the registers nor the issue
// slots for a long cache (65,536 candidates of one head in one work group: 84 us).
//   count   each slice's histogram of the top 11 bits
//   edge    the bin of the smallest kept key, from all slices' histograms; the
//           candidates in it go into one list, in any order
//   write   the exact edge from the list (every slice for itself), and the kept
//           positions at the place that the counts of the slices before give
// Bound by the launches and by what each waits for (65,537 positions of 2 heads:
// 4.6, 9.4 and 11.7 us, the copy 5.1; 28.6 us in all, 3.6 for the bytes).
constexpr int SL_T = 256, SL_V = 16, SL_N = SL_T * SL_V;

struct EvictLong {
  uint16_t* hist;  // [pair][slice][EV_BINS]
  int* before;     // [pair][slice]: kept in earlier slices by the first 11 bits alone
  int* n_list;     // [pair]
  int* need;       // [pair]: how many of the list are kept
  uint2* list;     // [pair][slices * SL_N]: (key, position)
  int slices;
};

template <int STEP>
__global__ void __launch_bounds__(SL_T) k_evict_long(PagedView kv, BatchView bt, int budget, int first, int recent, const EvictLong g,
                                                     int* __restrict__ kept, int* __restrict__ dst_lens) {
  __shared__ int hist[EV_BINS];
  __shared__ int s_wave[1][SL_T / 64];
  __shared__ Edge s_edge;
  __shared__ int s_sum[3];
  const int slice = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int64_t pair = static_cast<int64_t>(b) * kv.n_kv_heads + h;
  const int len = seq_len(bt, kv, b);
  int* out = kept + pair * budget;
  if constexpr (STEP == 0) {
    if (slice == 0 && tid == 0) g.n_list[pair] = 0;
    if (slice == 0 && h == 0 && tid == 0) dst_lens[b] = min(len, budget);
    kept_ends(len, budget, first, recent, slice * SL_T + tid, g.slices * SL_T, out);
  }
  if (len <= budget || budget - first - recent == 0) return;
  const int begin = first & ~(SL_V - 1), end = len - recent;
  const int n_slices = (end - begin + SL_N - 1) / SL_N;
  if (slice >= n_slices) return;
  const int j0 = begin + slice * SL_N + tid * SL_V;
  unsigned key[SL_V];
  load_keys<SL_V>(kv, bt, b, h, j0, end, key);
  auto candidate = [&](int i) { return j0 + i >= first && j0 + i < end; };
  auto clear = [&] {
    for (int i = tid; i < EV_BINS; i += SL_T) hist[i] = 0;
    if (tid < 3) s_sum[tid] = 0;
    __syncthreads();
  };
  constexpr int PER = EV_BINS / SL_T;
  uint16_t* mine = g.hist + (pair * g.slices + slice) * EV_BINS;
  uint2* list = g.list + pair * g.slices * SL_N;
  if constexpr (STEP == 0) {
    clear();
#pragma unroll
    for (int i = 0; i < SL_V; ++i)
      if (candidate(i)) atomicAdd(&hist[key[i] >> 21], 1);
    __syncthreads();
    uint32_t w[PER / 2];
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) w[i] = static_cast<uint32_t>(hist[tid * PER + 2 * i]) | static_cast<uint32_t>(hist[tid * PER + 2 * i + 1]) << 16;
    *reinterpret_cast<u32x4*>(mine + tid * PER) = u32x4{w[0], w[1], w[2], w[3]};
  } else if constexpr (STEP == 1) {
    clear();
    int sum[PER] = {}, before[PER] = {};  // of all slices, and of those before this one
    const uint16_t* other = g.hist + pair * g.slices * EV_BINS + tid * PER;
#pragma unroll 4
    for (int s = 0; s < n_slices; ++s) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(other + static_cast<int64_t>(s) * EV_BINS);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = w[i / 2] >> (16 * (i % 2)) & 0xffff;
        sum[i] += c;
        before[i] += s < slice ? c : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) hist[tid * PER + i] = sum[i];
    __syncthreads();
    find_edge<PER>(hist, EV_BINS, budget - first - recent, s_wave, &s_edge);
    const unsigned bin = s_edge.bin;
    int above = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) above += tid * PER + i > static_cast<int>(bin) ? before[i] : 0;
    int n[1] = {above}, all[1];
    block_prefix(n, s_wave, all);
    if (tid == 0) g.before[pair * g.slices + slice] = all[0];
    if (tid == 0 && slice == 0) g.need[pair] = s_edge.need;
    n[0] = 0;
#pragma unroll
    for (int i = 0; i < SL_V; ++i) n[0] += candidate(i) && key[i] >> 21 == bin;
    block_prefix(n, s_wave, all);
    if (tid == 0) s_sum[0] = all[0] ? atomicAdd(&g.n_list[pair], all[0]) : 0;
    __syncthreads();
    int o = s_sum[0] + n[0];
#pragma unroll
    for (int i = 0; i < SL_V; ++i)
      if (candidate(i) && key[i] >> 21 == bin) list[o++] = make_uint2(key[i], j0 + i);
  } else {
    // The list, in registers as far as OWN entries a lane go.
    constexpr int OWN = 16;
    const int n_list = g.n_list[pair];
    int need = g.need[pair];
    uint2 own[OWN];
#pragma unroll
    for (int k = 0; k < OWN; ++k) own[k] = list[min(tid + k * SL_T, n_list - 1)];
    auto members = [&](const auto& f) {
#pragma unroll
      for (int k = 0; k < OWN; ++k)
        if (tid + k * SL_T < n_list) f(own[k]);
      for (int i = tid + OWN * SL_T; i < n_list; i += SL_T) f(list[i]);
    };
    unsigned edge = list[0].x & ~0u << 21;
#pragma unroll 1
    for (int pass = 1; pass < 3; ++pass) {
      const int shift = pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : EV_BINS;
      const unsigned mask = pass == 1 ? ~0u << 21 : ~0u << 10;
      clear();
      members([&](const uint2& x) {
        if ((x.x & mask) == edge) atomicAdd(&hist[(x.x >> shift) & (bins - 1)], 1);
      });
      __syncthreads();
      find_edge<PER>(hist, EV_BINS, need, s_wave, &s_edge);
      edge |= static_cast<unsigned>(s_edge.bin) << shift;
      need = s_edge.need;
    }
    // members of earlier slices: larger ones, equal ones
    int c[2] = {0, 0};
    const int slice_begin = begin + slice * SL_N;
    members([&](const uint2& x) {
      if (static_cast<int>(x.y) < slice_begin) {
        c[0] += x.x > edge;
        c[1] += x.x == edge;
      }
    });
    if (c[0]) atomicAdd(&s_sum[0], c[0]);
    if (c[1]) atomicAdd(&s_sum[1], c[1]);
    __syncthreads();
    const int larger = s_sum[0], equal = s_sum[1];
    int n[1] = {0}, all[1];
#pragma unroll
    for (int i = 0; i < SL_V; ++i) n[0] += candidate(i) && key[i] == edge;
    block_prefix(n, s_wave, all);
    int rank = equal + n[0];
    unsigned keep = 0;
#pragma unroll
    for (int i = 0; i < SL_V; ++i)
      if (candidate(i) && (key[i] > edge || (key[i] == edge && rank++ < need))) keep |= 1u << i;
    n[0] = __popc(keep);
    block_prefix(n, s_wave, all);
    int o = first + g.before[pair * g.slices + slice] + larger + min(equal, need) + n[0];
#pragma unroll
    for (int i = 0; i < SL_V; ++i)
      if (keep >> i & 1) out[o++] = j0 + i;
  }
}

// A lane copies 16 bytes of a kept row, of k or of v (8 x 8 lists of 1024 rows of 64
// halves, 33.6 MB read and written: 7.3 us, 4.6 TB/s).
__global__ void __launch_bounds__(256) k_evict_copy(PagedView kv, BatchView bt, int esz, int budget,
                                                    const int* __restrict__ dst_pages, int max_dst_pages,
                                                    const int* __restrict__ kept) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int per = kv.hd * esz / 16;  // 16-byte pieces of a row
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t i64 = c / (2 * per);
  if (i64 >= budget) return;
  const int i = static_cast<int>(i64), piece = static_cast<int>(c - i64 * (2 * per));
  const int src = kept[(static_cast<int64_t>(b) * kv.n_kv_heads + h) * budget + i];
  if (src < 0 || (i >> kv.page_shift) >= max_dst_pages) return;
  const int sp = page_of(bt, kv, b, src);
  const int dp = dst_pages[static_cast<int64_t>(b) * max_dst_pages + (i >> kv.page_shift)];
  if (sp < 0 || static_cast<unsigned>(dp) >= static_cast<unsigned>(kv.n_pages)) return;
  char* base = piece < per ? kv.k : kv.v;
  const int64_t o = static_cast<int64_t>(piece < per ? piece : piece - per) * 16;
  *reinterpret_cast<u32x4*>(base + elem_of(kv, dp, i, h) * esz + o) =
      *reinterpret_cast<const u32x4*>(base + elem_of(kv, sp, src, h) * esz + o);
  if (piece == 0) *weight_of(kv, dp, i, h) = *weight_of(kv, sp, src, h);
}

template <typename TC, typename TI>
void append(const PagedView& kv, const BatchView& bt, const void* k, const void* v, int64_t kv_stride, void* q,
            int64_t q_stride, int n_heads, float rope_base, int slices, hipStream_t s) {
  const bool rotate = rope_base > 0.0f;
  hipLaunchKernelGGL((k_paged_append<TC, TI>), dim3(bt.n_rows, slices), dim3(256), 0, s, kv, bt,
                     static_cast<const TI*>(k), static_cast<const TI*>(v), kv_stride, static_cast<TI*>(q), q_stride,
                     n_heads, rotate ? log2(static_cast<double>(rope_base)) : 0.0, rotate ? 1 : 0);
}

}  // namespace

hipError_t launch_paged_append(const PagedView& kv, int kv_type, const BatchView& bt, int io_type, const void* k,
                               const void* v, int64_t kv_stride, void* q, int64_t q_stride, int n_heads,
                               float rope_base, int n_cu, hipStream_t s) {
  const int pieces = (2 * kv.n_kv_heads + (q ? n_heads : 0)) * (kv.hd / 8);
  int slices = (pieces + 255) / 256;
  while (slices > 1 && static_cast<int64_t>(bt.n_rows) * slices > 4 * n_cu) slices = (slices + 1) / 2;
  const bool f32 = io_type == MCPM_TYPE_F32;
  if (kv_type == MCPM_TYPE_F32) append<float, float>(kv, bt, k, v, kv_stride, q, q_stride, n_heads, rope_base, slices, s);
  else if (kv_type == MCPM_TYPE_F16 && f32) append<_Float16, float>(kv, bt, k, v, kv_stride, q, q_stride, n_heads, rope_base, slices, s);
  else if (kv_type == MCPM_TYPE_F16) append<_Float16, _Float16>(kv, bt, k, v, kv_stride, q, q_stride, n_heads, rope_base, slices, s);
  else if (f32) append<__bf16, float>(kv, bt, k, v, kv_stride, q, q_stride, n_heads, rope_base, slices, s);
  else append<__bf16, __bf16>(kv, bt, k, v, kv_stride, q, q_stride, n_heads, rope_base, slices, s);
  return hipGetLastError();
}

namespace {
constexpr int EV_MOST = 16 * EV_T;
// Positions from the first candidate's run of SL_V on, at most.
int evict_span(const BatchView& bt, int first, int recent) { return bt.max_len - recent - (first & ~(SL_V - 1)); }
}  // namespace

size_t paged_evict_scratch(const PagedView& kv, const BatchView& bt, int first, int recent) {
  const int n = evict_span(bt, first, recent);
  if (n <= EV_MOST) return 0;
  const size_t pairs = static_cast<size_t>(bt.n_seq) * kv.n_kv_heads, slices = (static_cast<size_t>(n) + SL_N - 1) / SL_N;
  return pairs * slices * (EV_BINS * sizeof(uint16_t) + SL_N * sizeof(uint2) + sizeof(int)) + 2 * pairs * sizeof(int);
}

hipError_t launch_paged_evict(const PagedView& kv, int kv_type, const BatchView& bt, int budget, int first, int recent,
                              const int* dst_pages, int max_dst_pages, int* kept, int* dst_lens, void* scratch, hipStream_t s) {
  const int esz = kv_type == MCPM_TYPE_F32 ? 4 : 2;
  const dim3 grid(kv.n_kv_heads, bt.n_seq);
  const int n = evict_span(bt, first, recent);
  if (n <= 4 * EV_T) {
    hipLaunchKernelGGL(k_evict_select<4>, grid, dim3(EV_T), 0, s, kv, bt, budget, first, recent, kept, dst_lens);
  } else if (n <= EV_MOST) {
    hipLaunchKernelGGL(k_evict_select<16>, grid, dim3(EV_T), 0, s, kv, bt, budget, first, recent, kept, dst_lens);
  } else {
    const int64_t pairs = static_cast<int64_t>(bt.n_seq) * kv.n_kv_heads;
    EvictLong g{};
    g.slices = (n + SL_N - 1) / SL_N;
    char* p = static_cast<char*>(scratch);
    g.hist = reinterpret_cast<uint16_t*>(p);
    p += pairs * g.slices * EV_BINS * sizeof(uint16_t);
    g.list = reinterpret_cast<uint2*>(p);
    p += pairs * g.slices * SL_N * sizeof(uint2);
    g.before = reinterpret_cast<int*>(p);
    g.n_list = g.before + pairs * g.slices;
    g.need = g.n_list + pairs;
    const dim3 slices(g.slices, kv.n_kv_heads, bt.n_seq);
    hipLaunchKernelGGL(k_evict_long<0>, slices, dim3(SL_T), 0, s, kv, bt, budget, first, recent, g, kept, dst_lens);
    hipLaunchKernelGGL(k_evict_long<1>, slices, dim3(SL_T), 0, s, kv, bt, budget, first, recent, g, kept, dst_lens);
    hipLaunchKernelGGL(k_evict_long<2>, slices, dim3(SL_T), 0, s, kv, bt, budget, first, recent, g, kept, dst_lens);
  }
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const int64_t lanes = static_cast<int64_t>(budget) * (2 * (kv.hd * esz / 16));
  hipLaunchKernelGGL(k_evict_copy, dim3(static_cast<unsigned>((lanes + 255) / 256), kv.n_kv_heads, bt.n_seq), dim3(256), 0, s, kv, bt,
                     esz, budget, dst_pages, max_dst_pages, kept);
  return hipGetLastError();
}

}  // namespace mcpm
