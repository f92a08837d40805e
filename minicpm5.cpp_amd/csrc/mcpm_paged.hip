// mcpm_paged.hip -- writing side of the paged cache: the append of new tokens
// (with the rotation of k and q) and the eviction by accumulated weight.
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
// the sine, and leave (cos, sin) in LDS.
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

// One work group per (sequence, kv head): the key of the smallest kept weight
// by four 8-bit histogram passes, then the kept positions in order.
__global__ void __launch_bounds__(EV_T) k_evict_select(PagedView kv, BatchView bt, int budget, int first, int recent,
                                                       int* __restrict__ kept, int* __restrict__ dst_lens) {
  __shared__ unsigned hist[256];
  __shared__ unsigned s_key, s_need;
  __shared__ int s_wave[2][EV_T / 64];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int len = seq_len(bt, kv, b);
  int* out = kept + (static_cast<int64_t>(b) * kv.n_kv_heads + h) * budget;
  const int n_keep = min(len, budget);
  if (h == 0 && tid == 0) dst_lens[b] = n_keep;
  for (int i = n_keep + tid; i < budget; i += EV_T) out[i] = -1;
  if (len <= budget) {
    for (int i = tid; i < len; i += EV_T) out[i] = i;
    return;
  }
  const int lo = first, hi = len - recent;  // candidates
  auto key_at = [&](int j) {
    const int page = page_of(bt, kv, b, j);
    return page < 0 ? 0u : weight_key(*weight_of(kv, page, j, h));
  };
  if (tid == 0) {
    s_key = 0;
    s_need = budget - first - recent;
  }
  __syncthreads();
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += EV_T) hist[i] = 0;
    __syncthreads();
    const unsigned pre = s_key, need = s_need;
    const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int j = lo + tid; j < hi; j += EV_T) {
      const unsigned key = key_at(j);
      if ((key & mask) == pre) atomicAdd(&hist[(key >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      unsigned left = need;
      int d = 255;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      s_key = pre | (static_cast<unsigned>(d) << shift);
      s_need = left;
    }
    __syncthreads();
  }
  const unsigned edge = s_key, need = s_need;  // kept: key > edge, and the first `need` that equal it
  int n_eq = 0, n_out = 0;
  for (int j0 = 0; j0 < len; j0 += EV_T) {
    const int j = j0 + tid;
    const bool in = j < len, mid = in && j >= lo && j < hi;
    const unsigned key = mid ? key_at(j) : 0u;
    const bool eq = mid && key == edge;
    const unsigned long long below = (1ull << lane) - 1;
    const unsigned long long me = __ballot(eq);
    if (lane == 0) s_wave[0][wv] = __popcll(me);
    __syncthreads();
    int rank = n_eq + __popcll(me & below);
    for (int w = 0; w < EV_T / 64; ++w) {
      if (w < wv) rank += s_wave[0][w];
      n_eq += s_wave[0][w];
    }
    const bool keep = in && (!mid || key > edge || (eq && rank < static_cast<int>(need)));
    const unsigned long long mk = __ballot(keep);
    if (lane == 0) s_wave[1][wv] = __popcll(mk);
    __syncthreads();
    int at = n_out + __popcll(mk & below);
    for (int w = 0; w < EV_T / 64; ++w) {
      if (w < wv) at += s_wave[1][w];
      n_out += s_wave[1][w];
    }
    if (keep && at < n_keep) out[at] = j;
  }
}

// A lane copies 16 bytes of a kept row, of k or of v.
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

hipError_t launch_paged_evict(const PagedView& kv, int kv_type, const BatchView& bt, int budget, int first, int recent,
                              const int* dst_pages, int max_dst_pages, int* kept, int* dst_lens, hipStream_t s) {
  const int esz = kv_type == MCPM_TYPE_F32 ? 4 : 2;
  hipLaunchKernelGGL(k_evict_select, dim3(kv.n_kv_heads, bt.n_seq), dim3(EV_T), 0, s, kv, bt, budget, first, recent, kept,
                     dst_lens);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const int64_t lanes = static_cast<int64_t>(budget) * (2 * (kv.hd * esz / 16));
  hipLaunchKernelGGL(k_evict_copy, dim3(static_cast<unsigned>((lanes + 255) / 256), kv.n_kv_heads, bt.n_seq), dim3(256), 0, s, kv, bt,
                     esz, budget, dst_pages, max_dst_pages, kept);
  return hipGetLastError();
}

}  // namespace mcpm
