// Log probability, rank and entropy of given tokens in their logit rows, with each row's top
// alternatives, for MI355X (gfx950).
//
// With m the row's maximum, S = sum e^(x - m) and T = sum (x - m) e^(x - m):
//   log p(t) = (x_t - m) - log S,  entropy = log S - T / S,
//   rank(t)  = 1 + #{columns before t in descending order, ties by ascending column}.
// One pass: a workgroup takes a slice of a row into registers and leaves its (m, S, T), the
// number of its columns before the token and its n first columns; a second launch, one
// workgroup per row, joins them.  S and T are float64 sums: next to a dominant token the
// entropy is what is left of S after 1, which float32 sums would lose.
//
// The n first columns of a slice are taken without a sort: the n-th largest of the 256
// threads' largest columns is a lower bound that at least n columns reach, and only threads
// whose largest reaches it hold such columns, so at most n times a thread's columns are left
// to be ranked against each other (a few more than n in practice).

#include "vocab_rows.h"

#include "rlt_mi355x.h"

#include <math.h>

namespace {

using namespace vocab;

constexpr int kMaxTop = 64;
constexpr int kMaxVocab = 1 << 20;
constexpr int kWideEpt = 32, kNarrowEpt = 8;  // columns per thread of a slice
constexpr int kList = kMaxTop * kWideEpt;     // columns that reach the bound, at most

struct SliceStat {
  double s, t;
  float m;
  uint32_t before;
};

struct LogprobParams {
  const void* logits;
  int64_t row_stride;   // elements
  int64_t num_rows, vocab;
  const int64_t* rows;  // nullptr: row i of the call is logit row i
  const int64_t* tokens;
  int64_t count;
  int top_n;
  int slices, ept;
  SliceStat* stats;               // [count][slices]
  unsigned long long* candidates;  // [count][slices][top_n]
  float* logprob;
  int64_t* rank;
  float* entropy;
  float* top_logprob;
  int64_t* top_tokens;
};

struct TopShared {
  unsigned long long best[kThreads];
  unsigned long long list[kList];
  unsigned long long bound;
  int count;
};

// The n largest of the workgroup's composites (item(i), i < items, of every thread) go to
// out(rank, composite); ranks without a composite get 0.
template <int ITEMS, class Item, class Out>
__device__ __forceinline__ void select_top(TopShared& sh, int n, int items, Item item, Out out) {
  const int t = threadIdx.x;
  unsigned long long best = 0;
  if constexpr (ITEMS > 0) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const unsigned long long c = item(i);
      best = best > c ? best : c;
    }
  } else {
    for (int i = 0; i < items; ++i) {
      const unsigned long long c = item(i);
      best = best > c ? best : c;
    }
  }
  sh.best[t] = best;
  if (t == 0) {
    sh.bound = 1;  // fewer than n threads with a column: all columns
    sh.count = 0;
  }
  __syncthreads();
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < kThreads; ++i) above += sh.best[i] > best;
  if (best && above == n - 1) sh.bound = best;
  __syncthreads();
  const unsigned long long bound = sh.bound;
  auto take = [&](int i) {
    const unsigned long long c = item(i);
    if (c >= bound) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kList) sh.list[at] = c;
    }
  };
  if (best >= bound) {
    if constexpr (ITEMS > 0) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) take(i);
    } else {
      for (int i = 0; i < items; ++i) take(i);
    }
  }
  __syncthreads();
  const int found = min(sh.count, kList);
  for (int e = t; e < found; e += kThreads) {
    const unsigned long long c = sh.list[e];
    int r = 0;
    for (int i = 0; i < found; ++i) r += sh.list[i] > c;
    if (r < n) out(r, c);
  }
  for (int r = found + t; r < n; r += kThreads) out(r, 0ull);
}

__device__ __forceinline__ double block_sum(double x, double* sh) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, RLT_WAVE);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}
__device__ __forceinline__ float block_max(float x, float* sh) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, RLT_WAVE));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
  __syncthreads();
  return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}

__device__ __forceinline__ int64_t source_row(const LogprobParams& P, int64_t r) {
  const int64_t row = P.rows ? P.rows[r] : r;
  return row >= 0 && row < P.num_rows ? row : -1;
}

template <int DT, int EPT>
__global__ __launch_bounds__(kThreads) void rlt_logprob_slices_kernel(LogprobParams P) {
  __shared__ TopShared top;
  __shared__ double dsh[4];
  __shared__ float fsh[4];
  using S = Slice<DT, EPT>;
  constexpr int ELT = DT == RLT_F32 ? 4 : 2;
  const int64_t r = blockIdx.y;
  const int slice = blockIdx.x;
  const int64_t row = source_row(P, r);
  if (row < 0) return;
  const uint8_t* const src = (const uint8_t*)P.logits + row * P.row_stride * ELT;
  const int64_t begin = (int64_t)slice * EPT * kThreads;
  S x;
  x.load(src, begin, P.vocab);
  const int64_t token = P.tokens[r];
  unsigned long long mine = ~0ull;  // nothing comes before no token
  if (token >= 0 && token < P.vocab)
    mine = composite(order_key(load_as_f32<DT>(src, token)), (uint32_t)token);
  float m = -INFINITY;
  uint32_t before = 0;
#pragma unroll
  for (int i = 0; i < S::NP; ++i) {
    const int64_t c = S::column(begin, i);
#pragma unroll
    for (int e = 0; e < S::VE; ++e) {
      const bool ok = c + e < P.vocab;
      const float v = x.at(i, e);
      m = ok ? fmaxf(m, v) : m;
      before += ok && composite(order_key(v), (uint32_t)(c + e)) > mine;
    }
  }
  m = block_max(m, fsh);
  // e^d as 2^(d log2 e), the product's rounding made up for
  constexpr float kL2e = 1.4426950408889634f, kL2eLo = 1.925963033500011e-8f, kLn2 = 0.6931471805599453f;
  double s = 0.0, q = 0.0;
#pragma unroll
  for (int i = 0; i < S::NP; ++i) {
    const int64_t c = S::column(begin, i);
#pragma unroll
    for (int e = 0; e < S::VE; ++e) {
      const float d = x.at(i, e) - m;
      const float hi = d * kL2e;
      const float lo = __builtin_fmaf(d, kL2eLo, __builtin_fmaf(d, kL2e, -hi));
      const float y = __builtin_amdgcn_exp2f(hi);
      float w = __builtin_fmaf(y, lo * kLn2, y);
      // columns past the row weigh nothing, nor do masked logits: -inf, and finite ones so far
      // down that hi or lo overflow
      if (!(c + e < P.vocab) || x.at(i, e) == -INFINITY || hi < -160.f) w = 0.f;
      s += (double)w;
      q += w == 0.f ? 0.0 : (double)w * (double)d;
    }
  }
  s = block_sum(s, dsh);
  q = block_sum(q, dsh);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) before += __shfl_xor(before, o, RLT_WAVE);
  __syncthreads();
  uint32_t* const counts = (uint32_t*)fsh;
  if ((threadIdx.x & 63) == 0) counts[threadIdx.x >> 6] = before;
  __syncthreads();
  if (threadIdx.x == 0) {
    SliceStat st;
    st.s = s;
    st.t = q;
    st.m = m;
    st.before = counts[0] + counts[1] + counts[2] + counts[3];
    P.stats[r * P.slices + slice] = st;
  }
  if (P.top_n > 0) {
    unsigned long long* const dst = P.candidates + (r * P.slices + slice) * P.top_n;
    select_top<EPT>(
        top, P.top_n, EPT,
        [&](int k) {
          const int i = k / S::VE, e = k % S::VE;
          const int64_t c = S::column(begin, i) + e;
          return c < P.vocab ? composite(order_key(x.at(i, e)), (uint32_t)c) : 0ull;
        },
        [&](int rank, unsigned long long c) { dst[rank] = c; });
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void rlt_logprob_rows_kernel(LogprobParams P) {
  __shared__ TopShared top;
  __shared__ double dsh[4];
  __shared__ float fsh[4];
  constexpr int ELT = DT == RLT_F32 ? 4 : 2;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  const int64_t row = source_row(P, r);
  const float nan = __uint_as_float(0x7fc00000u);
  if (row < 0) {
    if (t == 0) {
      P.logprob[r] = P.entropy[r] = nan;
      P.rank[r] = 0;
    }
    for (int i = t; i < P.top_n; i += kThreads) {
      P.top_logprob[r * P.top_n + i] = nan;
      P.top_tokens[r * P.top_n + i] = -1;
    }
    return;
  }
  const SliceStat* const st = P.stats + r * P.slices;
  float m = -INFINITY;
  for (int i = t; i < P.slices; i += kThreads) m = fmaxf(m, st[i].m);
  m = block_max(m, fsh);
  double s = 0.0, q = 0.0, before = 0.0;
  for (int i = t; i < P.slices; i += kThreads) {
    const SliceStat x = st[i];
    before += x.before;
    if (x.m == -INFINITY && x.s == 0.0) continue;  // nothing but masked logits
    const double d = (double)x.m - (double)m, w = exp(d);
    s += x.s * w;
    q += (x.t + d * x.s) * w;
  }
  s = block_sum(s, dsh);
  q = block_sum(q, dsh);
  before = block_sum(before, dsh);
  const double lse = log(s);  // over the maximum; a row without a finite one gives NaN
  const bool ok = m > -INFINITY;
  if (t == 0) {
    const int64_t token = P.tokens[r];
    const bool in = token >= 0 && token < P.vocab;
    const uint8_t* const src = (const uint8_t*)P.logits + row * P.row_stride * ELT;
    P.logprob[r] = ok && in ? (float)(((double)load_as_f32<DT>(src, token) - (double)m) - lse) : nan;
    P.entropy[r] = ok ? (float)(lse - q / s) : nan;
    P.rank[r] = in ? 1 + (int64_t)before : 0;
  }
  if (P.top_n > 0) {
    const unsigned long long* const c = P.candidates + r * P.slices * P.top_n;
    const int total = P.slices * P.top_n, items = (total + kThreads - 1) / kThreads;
    select_top<0>(
        top, P.top_n, items,
        [&](int i) { return i * kThreads + t < total ? c[i * kThreads + t] : 0ull; },
        [&](int rank, unsigned long long x) {
          const int64_t at = r * P.top_n + rank;
          P.top_tokens[at] = x ? (int64_t)composite_col(x) : -1;
          P.top_logprob[at] =
              x && ok ? (float)(((double)key_value((uint32_t)(x >> 32)) - (double)m) - lse) : nan;
        });
  }
}

// Columns per thread: wide slices where they fill the chip (fewer candidates to join), narrow
// ones for a few rows, whose time is one slice's.
int slice_ept(int64_t count, int64_t vocab) {
  const int64_t wide = (vocab + kWideEpt * kThreads - 1) / (kWideEpt * kThreads);
  return count * wide < 256 && vocab <= 262144 ? kNarrowEpt : kWideEpt;
}
int64_t slices_of(int64_t count, int64_t vocab) {
  const int64_t w = (int64_t)slice_ept(count, vocab) * kThreads;
  return (vocab + w - 1) / w;
}

template <int DT>
void launch(const LogprobParams& P, hipStream_t stream) {
  const dim3 grid((unsigned)P.slices, (unsigned)P.count);
  if (P.ept == kWideEpt)
    hipLaunchKernelGGL((rlt_logprob_slices_kernel<DT, kWideEpt>), grid, dim3(kThreads), 0, stream, P);
  else
    hipLaunchKernelGGL((rlt_logprob_slices_kernel<DT, kNarrowEpt>), grid, dim3(kThreads), 0, stream, P);
  hipLaunchKernelGGL((rlt_logprob_rows_kernel<DT>), dim3((unsigned)P.count), dim3(kThreads), 0, stream, P);
}

}  // namespace

extern "C" {

size_t rlt_token_logprobs_workspace_size(int64_t count, int64_t vocab, int32_t top_n) {
  if (count <= 0 || vocab <= 0 || vocab > kMaxVocab || top_n < 0 || top_n > kMaxTop || count > 65535)
    return 0;
  const int64_t slices = slices_of(count, vocab);
  return (size_t)(count * slices) * (sizeof(SliceStat) + (size_t)top_n * sizeof(unsigned long long));
}

int rlt_token_logprobs(const void* logits, int32_t logits_dtype, int64_t row_stride,
                       int64_t num_rows, int64_t vocab, const int64_t* rows, const int64_t* tokens,
                       int64_t count, int32_t top_n, float* logprob, int64_t* rank, float* entropy,
                       float* top_logprob, int64_t* top_tokens, void* workspace,
                       size_t workspace_bytes, hipStream_t stream) {
  if (count < 0 || num_rows < 0 || vocab < 1 || top_n < 0 || (num_rows > 1 && row_stride < vocab) ||
      (!rows && count > num_rows))
    return RLT_ERR_ARGUMENT;
  if (logits_dtype != RLT_F32 && logits_dtype != RLT_BF16 && logits_dtype != RLT_F16)
    return RLT_ERR_UNSUPPORTED;
  if (vocab > kMaxVocab || top_n > kMaxTop || top_n > vocab || count > 65535) return RLT_ERR_UNSUPPORTED;
  if (count == 0) return RLT_OK;
  if ((!logits && num_rows > 0) || !tokens || !logprob || !rank || !entropy ||
      (top_n && (!top_logprob || !top_tokens)))
    return RLT_ERR_ARGUMENT;
  if (!workspace || (uintptr_t)workspace % 8 ||
      workspace_bytes < rlt_token_logprobs_workspace_size(count, vocab, top_n))
    return RLT_ERR_WORKSPACE;
  LogprobParams P;
  P.logits = logits;
  P.row_stride = row_stride;
  P.num_rows = num_rows;
  P.vocab = vocab;
  P.rows = rows;
  P.tokens = tokens;
  P.count = count;
  P.top_n = top_n;
  P.ept = slice_ept(count, vocab);
  P.slices = (int)slices_of(count, vocab);
  P.stats = (SliceStat*)workspace;
  P.candidates = (unsigned long long*)(P.stats + count * P.slices);
  P.logprob = logprob;
  P.rank = rank;
  P.entropy = entropy;
  P.top_logprob = top_logprob;
  P.top_tokens = top_tokens;
  switch (logits_dtype) {
    case RLT_F32: launch<RLT_F32>(P, stream); break;
    case RLT_BF16: launch<RLT_BF16>(P, stream); break;
    default: launch<RLT_F16>(P, stream); break;
  }
  return rlt_launch_status();
}

}  // extern "C"
