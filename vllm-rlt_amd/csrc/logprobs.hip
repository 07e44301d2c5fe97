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
// The n first columns of a slice are taken without a sort.  Bounds on the waves' lanes' largest
// columns give one that n columns of the slice reach; those that reach it (a few more than n)
// are listed wave by wave and ranked by counting.  Where ties or an uneven slice make a list too
// long, the bound is taken over all threads' largest (value, column) pairs, which are all
// different: then at most n threads hold such columns.
//
// The instructions of a column bound the kernel (160 rows of 49152 float32 columns with 20
// alternatives: 15 us for the slices, 2.1 TB/s, and 5 us to join them); of a workgroup's 9 us the
// loads take 1.6, the bound 1, the weights 0.8, the columns ahead 0.6, the listing and the ranks
// 1.3 each.  float64 sums cost more than the loads, so four weights at a time are added in
// float32 first; weights of exactly 1 (the maximum) are counted instead, and nothing is lost
// next to them.
//
// A weight's exponent and exponential are float32: with d = x - m it is off by at most
// (2 + 2.3 |d|) 2^-24 of itself, two float32 additions add 2 half steps, and log S is off by
// E[4 + 2.3 |d|] 2^-24, E the mean under the row's distribution.  Most of it averages out over the
// columns: 160 rows of 49152 come out as near to float64 (3e-8 of the values) as float32 torch code.

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
  uint2 wave_bound[kThreads / 64];  // of n, of n / 4
  int wave_count[kThreads / 64];
  int count;  // select_top
};

// Ranks the `found` different composites of sh.list by counting; out(rank, composite) for the
// first n, 0 behind the last.
template <class Out>
__device__ __forceinline__ void rank_list(const TopShared& sh, int found, int n, Out out) {
  for (int e = threadIdx.x; e < found; e += kThreads) {
    const unsigned long long c = sh.list[e];
    int r = 0;
#pragma unroll 8
    for (int i = 0; i < found; ++i) r += sh.list[i] > c;
    if (r < n) out(r, c);
  }
  for (int r = found + (int)threadIdx.x; r < n; r += kThreads) out(r, 0ull);
}

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
  rank_list(sh, min(sh.count, kList), n, out);
}

// Lower bounds that n and `part` of the wave's 64 values reach: the n-th largest, its low bits
// cleared (0: fewer than n are positive).  16-bit logits' keys have no low bits; a float32 one's
// bound lies up to 2^-9 below it, for half the steps.
__device__ __forceinline__ uint2 wave_nth(uint32_t x, int n, int part) {
  uint2 bound = make_uint2(0, 0);
#pragma unroll 6
  for (int bit = 31; bit >= 14; --bit) {
    const uint2 next = make_uint2(bound.x | (1u << bit), bound.y | (1u << bit));
    if (__popcll(__builtin_amdgcn_ballot_w64(x >= next.x)) >= n) bound.x = next.x;
    if (__popcll(__builtin_amdgcn_ballot_w64(x >= next.y)) >= part) bound.y = next.y;
  }
  return bound;
}

__device__ __forceinline__ int64_t source_row(const LogprobParams& P, int64_t r) {
  const int64_t row = P.rows ? P.rows[r] : r;
  return row >= 0 && row < P.num_rows ? row : -1;
}

// A lower bound that n columns of the workgroup reach: the threads' largest columns reach the
// least of the waves' bounds for n / 4, and the largest of their bounds for n (the better one
// where the row ends inside the first wave's columns).  Wave w's part, in LDS; the waves' lists
// are cleared (a barrier follows before they are used).
constexpr int kWaveList = 64;
__device__ __forceinline__ void put_bound(TopShared& sh, uint32_t largest, int n) {
  const uint2 bound = wave_nth(largest, n, (n + kThreads / 64 - 1) / (kThreads / 64));
  if ((threadIdx.x & 63) == 0) sh.wave_bound[threadIdx.x >> 6] = bound;
  sh.list[threadIdx.x] = 0;
}
__device__ __forceinline__ uint32_t get_bound(const TopShared& sh) {
  uint2 x = sh.wave_bound[0];
#pragma unroll
  for (int v = 1; v < kThreads / 64; ++v)
    x = make_uint2(max(x.x, sh.wave_bound[v].x), min(x.y, sh.wave_bound[v].y));
  return max(x.x, x.y);
}
// Columns that reach the bound go to their wave's list, without atomics; `count` is the same in
// every lane and goes on past a full list.
__device__ __forceinline__ void list_column(TopShared& sh, int& count, bool hit, unsigned long long c) {
  const uint64_t hits = __builtin_amdgcn_ballot_w64(hit);
  if (!hits) return;
  const int lane = threadIdx.x & 63;
  const int at = count + (int)__popcll(hits & ((1ull << lane) - 1));
  if (hit && at < kWaveList) sh.list[(threadIdx.x >> 6) * kWaveList + at] = c;
  count += (int)__popcll(hits);
}
// Ranks the waves' lists by counting; out(rank, composite) for the first n, 0 behind the last.
// False (of every thread alike): a list is not complete.
template <class Out>
__device__ __forceinline__ bool rank_lists(const TopShared& sh, int n, Out out) {
  const int t = threadIdx.x, lane = t & 63;
  int counts[kThreads / 64], found = 0, longest = 0;
#pragma unroll
  for (int v = 0; v < kThreads / 64; ++v) {
    counts[v] = sh.wave_count[v];
    found += counts[v];
    longest = max(longest, counts[v]);
  }
  if (longest > kWaveList) return false;
  if (lane < sh.wave_count[t >> 6]) {
    const unsigned long long c = sh.list[t];
    int r = 0;
#pragma unroll
    for (int v = 0; v < kThreads / 64; ++v)
      for (int i = 0; i < counts[v]; i += 8)  // (zeros behind a list's end)
#pragma unroll
        for (int k = 0; k < 8; ++k) r += sh.list[v * kWaveList + i + k] > c;
    if (r < n) out(r, c);
  }
  for (int r = found + t; r < n; r += kThreads) out(r, 0ull);
  return true;
}

// The next lower number; of -inf NaN, which nothing lies at or below.
__device__ __forceinline__ float below(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 is 0)
  if (b == 0xff800000u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(b == 0 ? 0x80000001u : b & 0x80000000u ? b + 1 : b - 1);
}

// A slice's statistics and first columns.  FULL: no column of it lies past the row.
template <int DT, int EPT, bool FULL>
__device__ __forceinline__ void scan_slice(const LogprobParams& P, const uint8_t* src, int64_t r, int slice, int token,
                                           TopShared& top, double (&sums)[kThreads / 64][2],
                                           uint32_t (&counts)[kThreads / 64][2], float (&maxima)[kThreads / 64]) {
  using S = Slice<DT, EPT>;
  const int t = threadIdx.x, w = t >> 6;
  const int begin = slice * EPT * kThreads, vocab = (int)P.vocab;
  S x;
  x.load(src, begin, FULL ? begin + EPT * kThreads : vocab);
  auto column = [&](int i) { return (int)S::column(begin, i); };
  auto inside = [&](int c) { return FULL || c < vocab; };
  const float xt = load_as_f32<DT>(src, token);
  // columns past the row become -inf, which weighs nothing
  if (!FULL) {
#pragma unroll
    for (int i = 0; i < S::NP; ++i)
#pragma unroll
      for (int e = 0; e < S::VE; ++e)
        if (column(i) + e >= vocab) x.set(i, e, -INFINITY);
  }
  float m = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < S::NP; ++i)
#pragma unroll
    for (int e = 0; e < S::VE; e += 2) {
      const float v0 = x.at(i, e), v1 = x.at(i, e + 1);
      m = fmaxf(fmaxf(m, v0), v1);
      nan |= __builtin_isunordered(v0, v1);
    }
  // the thread's largest column (NaN comes first; 0: none above -inf)
  const uint32_t mine = nan ? 0xffffffffu : m == -INFINITY ? 0u : order_key(m);
  m = wave_max(m);
  const float wave_top = m;
  if (P.top_n > 0) put_bound(top, mine, P.top_n);
  if ((t & 63) == 0) maxima[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(maxima[0], maxima[1]), fmaxf(maxima[2], maxima[3]));
  // (a slice without a finite maximum counts no ones: +inf or NaN spoils its sums, and with
  // nothing but -inf they are 0)
  const float from = m == -INFINITY ? 0.f : m;
  constexpr float kL2e = 1.4426950408889634f;
  double s = 0.0, q = 0.0;
  uint32_t ones = 0, before = 0;
  // (the instructions of a column bound the kernel: the maximum is looked for in its wave only)
  auto weigh = [&](auto counted) {
#pragma unroll
    for (int i = 0; i < S::NP; ++i)
#pragma unroll
      for (int f = 0; f < S::VE; f += 4) {
        float ws[4], qs[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float d = x.at(i, f + k) - from;
          float z = __builtin_amdgcn_exp2f(d * kL2e);
          if constexpr (decltype(counted)::value) {
            const bool one = d == 0.f;
            z = one ? 0.f : z;
            ones += one ? 1u : 0u;
          }
          ws[k] = z;
          qs[k] = z * fmaxf(d, -200.f);  // (d may be -inf where z is 0)
        }
        s += (double)((ws[0] + ws[1]) + (ws[2] + ws[3]));
        q += (double)((qs[0] + qs[1]) + (qs[2] + qs[3]));
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  if (wave_top == m && fabsf(m) < INFINITY) weigh(std::true_type{});
  else weigh(std::false_type{});
  // Columns ahead of the token: greater (or NaN), or equal in an earlier column.  A slice
  // before the token's takes "not below the token's" as "above the next lower number" (for
  // -inf: everything), one behind it "above"; the token's own looks at the columns.
  const int end = begin + EPT * kThreads;
  if (xt != xt) {
    // (of a NaN token, the NaN columns before it)
#pragma unroll
    for (int i = 0; i < S::NP; ++i)
#pragma unroll
      for (int e = 0; e < S::VE; ++e) {
        const float v = x.at(i, e);
        before += ((v != v) & (column(i) + e < token)) ? 1u : 0u;
      }
  } else if (token >= begin && token < end) {
#pragma unroll
    for (int i = 0; i < S::NP; ++i)
#pragma unroll
      for (int e = 0; e < S::VE; ++e) {
        const float v = x.at(i, e);
        before += ((!(v <= xt)) | ((v == xt) & (column(i) + e < token))) ? 1u : 0u;
      }
  } else {
    const float least = token >= end ? below(xt) : xt;
#pragma unroll
    for (int i = 0; i < S::NP; ++i)
#pragma unroll
      for (int e = 0; e < S::VE; ++e) before += !(x.at(i, e) <= least) ? 1u : 0u;
  }
  s = wave_sum(s);
  q = wave_sum(q);
  const uint32_t both = wave_sum(before << 16 | ones);  // (at most 64 EPT of each)
  if ((t & 63) == 0) {
    sums[w][0] = s;
    sums[w][1] = q;
    counts[w][0] = both >> 16;
    counts[w][1] = both & 0xffffu;
  }
  if (P.top_n > 0) {
    // (bound 0, fewer than n columns above -inf in each wave: every column reaches it, as any
    // does not lie below the NaN that is its value)
    const uint32_t bound = get_bound(top);
    const float least = key_value(bound);
    int listed = 0;
    if (__builtin_amdgcn_ballot_w64(mine >= bound) != 0) {
#pragma unroll
      for (int i = 0; i < S::NP; ++i)
#pragma unroll
        for (int e = 0; e < S::VE; ++e) {
          const int c = column(i) + e;
          const float v = x.at(i, e);
          list_column(top, listed, (!(v < least)) & inside(c), composite(order_key(v), (uint32_t)c));
        }
    }
    if ((t & 63) == 0) top.wave_count[w] = listed;
  }
  __syncthreads();
  if (t == 0) {
    SliceStat st;
    st.s = ((sums[0][0] + sums[1][0]) + (sums[2][0] + sums[3][0])) +
           (double)(counts[0][1] + counts[1][1] + counts[2][1] + counts[3][1]);
    st.t = (sums[0][1] + sums[1][1]) + (sums[2][1] + sums[3][1]);
    st.m = m;
    st.before = counts[0][0] + counts[1][0] + counts[2][0] + counts[3][0];
    P.stats[r * P.slices + slice] = st;
  }
  if (P.top_n > 0) {
    unsigned long long* const dst = P.candidates + (r * P.slices + slice) * P.top_n;
    auto put = [&](int rank, unsigned long long c) { dst[rank] = c; };
    if (!rank_lists(top, P.top_n, put)) {
      __syncthreads();
      select_top<EPT>(
          top, P.top_n, EPT,
          [&](int k) {
            const int c = column(k / S::VE) + k % S::VE;
            return inside(c) ? composite(order_key(x.at(k / S::VE, k % S::VE)), (uint32_t)c) : 0ull;
          },
          put);
    }
  }
}

template <int DT, int EPT>
__global__ __launch_bounds__(kThreads, EPT == kWideEpt ? 4 : 8) void rlt_logprob_slices_kernel(LogprobParams P) {
  __shared__ TopShared top;
  __shared__ double sums[kThreads / 64][2];
  __shared__ uint32_t counts[kThreads / 64][2];
  __shared__ float maxima[kThreads / 64];
  const int64_t r = blockIdx.y;
  const int slice = blockIdx.x;
  const int64_t wanted = P.tokens[r];
  const int64_t row = source_row(P, r);
  if (row < 0) return;
  const int token = wanted >= 0 && wanted < P.vocab ? (int)wanted : 0;
  const uint8_t* const src = (const uint8_t*)P.logits + row * P.row_stride * (DT == RLT_F32 ? 4 : 2);
  if ((int64_t)(slice + 1) * EPT * kThreads <= P.vocab)
    scan_slice<DT, EPT, true>(P, src, r, slice, token, top, sums, counts, maxima);
  else
    scan_slice<DT, EPT, false>(P, src, r, slice, token, top, sums, counts, maxima);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void rlt_logprob_rows_kernel(LogprobParams P) {
  __shared__ TopShared top;
  __shared__ double sh[2];  // the row's maximum, and the log of its sum over it
  constexpr int ELT = DT == RLT_F32 ? 4 : 2;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  const float nan = __uint_as_float(0x7fc00000u);
  // (the partial results of a row index outside the logits were not written: read for nothing)
  const unsigned long long* const c = P.candidates + r * P.slices * P.top_n;
  const int total = P.slices * P.top_n, items = (total + kThreads - 1) / kThreads;
  auto item = [&](int i) { return i * kThreads + t < total ? c[i * kThreads + t] : 0ull; };
  unsigned long long best = 0;
  for (int i = 0; i < items; ++i) best = max(best, item(i));
  const int64_t row = source_row(P, r);
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
  if (t < 64) {
    // one wave joins the slices while the others wait with their candidates
    const SliceStat* const st = P.stats + r * P.slices;
    const int64_t token = P.tokens[r];
    const bool in = token >= 0 && token < P.vocab;
    const float xt = load_as_f32<DT>((const uint8_t*)P.logits + row * P.row_stride * ELT, in ? token : 0);
    float m = -INFINITY;
    for (int i = t; i < P.slices; i += 64) m = fmaxf(m, st[i].m);
    m = wave_max(m);
    double s = 0.0, q = 0.0;
    uint32_t before = 0;
    for (int i = t; i < P.slices; i += 64) {
      const SliceStat x = st[i];
      before += x.before;
      if (x.m == -INFINITY && x.s == 0.0) continue;  // nothing but masked logits
      const double d = (double)x.m - (double)m, w = exp(d);
      s += x.s * w;
      q += (x.t + d * x.s) * w;
    }
    s = wave_sum(s);
    q = wave_sum(q);
    before = wave_sum(before);
    const double lse = log(s);  // over the maximum; a row without a finite one gives NaN
    if (t == 0) {
      const bool ok = m > -INFINITY;
      sh[0] = ok ? (double)m : (double)nan;
      sh[1] = lse;
      P.logprob[r] = ok && in ? (float)(((double)xt - (double)m) - lse) : nan;
      P.entropy[r] = ok ? (float)(lse - q / s) : nan;
      P.rank[r] = in ? 1 + (int64_t)before : 0;
    }
  }
  if (P.top_n > 0) {
    // (a candidate's key is 0 where a slice had fewer columns)
    put_bound(top, (uint32_t)(best >> 32), P.top_n);
    __syncthreads();
    const uint32_t bound = max(get_bound(top), 1u);
    int listed = 0;
    if (__builtin_amdgcn_ballot_w64((uint32_t)(best >> 32) >= bound) != 0)
      for (int i = 0; i < items; ++i) {
        const unsigned long long x = item(i);
        list_column(top, listed, (uint32_t)(x >> 32) >= bound, x);
      }
    if ((t & 63) == 0) top.wave_count[t >> 6] = listed;
    __syncthreads();
    const double m = sh[0], lse = sh[1];
    auto put = [&](int rank, unsigned long long x) {
      const int64_t at = r * P.top_n + rank;
      P.top_tokens[at] = x ? (int64_t)composite_col(x) : -1;
      P.top_logprob[at] = x ? (float)(((double)key_value((uint32_t)(x >> 32)) - m) - lse) : nan;
    };
    if (!rank_lists(top, P.top_n, put)) {
      __syncthreads();
      select_top<0>(top, P.top_n, items, item, put);
    }
  }
}

// Columns per thread: wide slices where they fill the chip (less to join, and a slice's fixed
// phases over more columns: 160 rows of 49152 columns 15.0 + 4.9 us, 19.7 + 5.7 in narrow
// ones), narrow ones for a few rows, whose time is one slice's (4 rows of 151936 bf16 columns
// 6.2 + 5.8 us, 8.2 + 4.6 in wide ones).
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
