// Acceptance along a tree of drafted tokens, greedy and sampled, for MI355X (gfx950).
//
// Node 0 of a request is its last committed token, node j + 1 draft j, whose parent is an
// earlier node.  Both walks start at node 0 and end where no child is accepted.  A child has
// a larger index than its parent and siblings come in index order, so one scan of the drafts
// in index order is the whole walk.
//
// Greedy: the child that holds the node's argmax token (the first, of several).  All logit
// rows' argmaxes are formed by row slices (the targets are an output), then one workgroup per
// request joins its slices and walks.  The logits' bytes bound it (32 requests of 32 nodes, 49152
// float32 columns: 31 us for 201 MB, 6.5 TB/s, and 5.4 to join); for one request the two
// launches (4.6 + 3.8 us).
//
// Sampled: at a node the children are tried in order, each drawn from the draft distribution
// q of the node.  With y the weights left of the target distribution p (at first y = p) and
// R = sum y (p counts as 1), a child of token t is accepted when u R q(t) < y(t); a rejected
// one leaves y' = max(y - R q, 0).  Since y only shrinks where it is positive, after k
// rejections y = max(p - C q, 0) with C = R_0 + .. + R_(k-1): no residual is stored, and a
// rejection costs one sum over the node's two rows.  Where no child is left the next token is
// drawn from y by inverse CDF.  The emitted tokens follow p whatever q and the tree are.
// C is the sum of two floats (48 bits).  A column's y is float32, from two fused steps with them:
// exact in sign and off by at most 2 half steps, 2^-23 of itself.  Four of them are added in
// float32 (two more half steps), these sums in float64: R and the CDF's coarse table are off by
// at most 2^-22 of themselves and C's 2^-48.  float64 weights took 1.7x the instructions that a
// pass is bound by.  Inside the drawn segment, and for a draft's own column, weights are float64.
//
// One workgroup per request, each wave 1024 columns at a time.  A node's first pass is bound by
// the rows' bytes: 83 GB/s of one CU, 6.6 TB/s of the chip at 128 requests.  It keeps what fits of
// the two rows on the CU: 4 steps (32768 columns) in registers and 2 in LDS, so that each
// further pass at the node costs 2.2 us at 49152 columns instead of 4.7.  The wave sums of the
// last pass are the CDF's coarse table.
// Measured: 4 requests, 49152 columns 15 us; 128 requests, 65536 columns, up to five passes 36.6 us
// (rereading the rows in every pass: 50).

#include "vocab_rows.h"

#include "rlt_mi355x.h"

#include <math.h>

namespace {

using namespace vocab;

constexpr int kMaxDrafts = 255;
constexpr int64_t kMaxVocab = 1 << 20;
constexpr int kSliceEpt = 32;
constexpr int64_t kMaxRequests = 1 << 22;  // of a sampled round: a launch's threads fit 32 bits
constexpr int64_t kMaxLaunch = UINT32_MAX;  // threads of a launch along one axis

// ---------------------------------------------------------------- greedy

template <int DT>
__global__ __launch_bounds__(kThreads) void rlt_tree_argmax_kernel(const void* logits, int64_t row_stride,
                                                                  int64_t vocab, int slices,
                                                                  unsigned long long* best) {
  __shared__ unsigned long long sh[4];
  using S = Slice<DT, kSliceEpt>;
  constexpr int ELT = DT == RLT_F32 ? 4 : 2;
  const int64_t row = blockIdx.x / slices;
  const int slice = (int)(blockIdx.x % slices);
  const int64_t begin = (int64_t)slice * kSliceEpt * kThreads;
  S x;
  x.load((const uint8_t*)logits + row * row_stride * ELT, begin, vocab);
  // columns ascend within a thread: the first of the largest keys
  uint32_t key = 0, at = 0;
#pragma unroll
  for (int i = 0; i < S::NP; ++i) {
    const int64_t c = S::column(begin, i);
#pragma unroll
    for (int e = 0; e < S::VE; ++e) {
      const uint32_t k = c + e < vocab ? order_key(x.at(i, e)) : 0u;
      at = k > key ? (uint32_t)(c + e) : at;
      key = k > key ? k : key;
    }
  }
  unsigned long long m = wave_max(key ? composite(key, at) : 0ull);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 4; ++i) m = sh[i] > m ? sh[i] : m;
    best[blockIdx.x] = m;
  }
}

__global__ __launch_bounds__(kThreads) void rlt_greedy_tree_kernel(
    const unsigned long long* best, int slices, const int64_t* draft_tokens, const int64_t* parents,
    const int64_t* drafts, int width, int64_t* targets, int64_t* path, int64_t* accepted,
    int64_t* next_token) {
  __shared__ int64_t target[kMaxDrafts + 1];
  __shared__ int walk[kMaxDrafts + 1];
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, nodes = width + 1;
  // node i's argmax: one lane group of 16 per node
  for (int i = t >> 4; i < nodes; i += kThreads / 16) {
    unsigned long long m = 0;
    for (int s = t & 15; s < slices; s += 16) {
      const unsigned long long c = best[(r * nodes + i) * slices + s];
      m = c > m ? c : m;
    }
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
      const unsigned long long c = __shfl_xor(m, o, RLT_WAVE);
      m = c > m ? c : m;
    }
    if ((t & 15) == 0) {
      target[i] = composite_col(m);
      targets[r * nodes + i] = target[i];
    }
  }
  __syncthreads();
  if (t >= 64) return;
  // one wave walks: lane holds drafts lane, lane + 64, ..
  const int64_t d = drafts[r];
  const int live = (int)(d < 0 ? 0 : d > width ? width : d);
  int64_t token[4], parent[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int j = lane + 64 * k;
    token[k] = j < live ? draft_tokens[r * width + j] : -1;
    parent[k] = j < live ? parents[r * width + j] : -1;
  }
  int node = 0, count = 0;
  for (;;) {
    int next = -1;
#pragma unroll
    for (int k = 3; k >= 0; --k) {
      // (a child comes after its parent: a larger index)
      const bool hit = lane + 64 * k >= node && parent[k] == node && token[k] == target[node];
      const uint64_t b = __builtin_amdgcn_ballot_w64(hit);
      if (b) next = 64 * k + __builtin_ctzll(b);
    }
    if (next < 0) break;
    node = next + 1;
    ++count;
    if (lane == 0) walk[count] = node;
  }
  if (lane == 0) walk[0] = 0;
  __builtin_amdgcn_wave_barrier();
  for (int i = lane; i < nodes; i += 64) path[r * nodes + i] = i <= count ? walk[i] : -1;
  if (lane == 0) {
    accepted[r] = count;
    next_token[r] = target[node];
  }
}

// ---------------------------------------------------------------- sampled

constexpr int kAccThreads = 512;
constexpr int kAccWaves = kAccThreads / 64;
constexpr int kRun = 16;                           // columns of a thread and step
constexpr int64_t kStep = (int64_t)kAccThreads * kRun;
constexpr int kHeldSteps = 4, kLdsSteps = 2;         // of a node's rows, kept for its further passes
constexpr int kMaxSegments = (int)(kMaxVocab / kStep) * kAccWaves;

struct __attribute__((packed, aligned(4))) Quad {
  float v[4];
};

struct AcceptShared {
  float4 kept[kLdsSteps][2][kRun / 4][kAccThreads];  // p and q of the steps from kHeldSteps on
  double seg[2][kMaxSegments];  // passes in turn: weight of every wave's kRun * 64 columns, in column order
  float px[kMaxDrafts], qx[kMaxDrafts], u[kMaxDrafts];
  int32_t parent[kMaxDrafts];
  int64_t token[kMaxDrafts];
  int32_t walk[kMaxDrafts + 1];  // the accepted path
  int64_t last;
};

// C as the two floats that a column's weight is formed with.  With no bit of it past them a float32
// weight and a float64 one have the same sign: where p - C q cancels, p - c_hi q is exact.  A segment
// that weighs anything then holds a column that does.
__device__ __forceinline__ double two_floats(double C) {
  const float hi = (float)C;
  return (double)hi + (double)(float)(C - (double)hi);
}

// y = max(p - C q, 0); NaN becomes 0 here and is looked for apart
__device__ __forceinline__ double left_of(float p, float q, double C) {
  return fmax(__builtin_fma(-C, (double)q, (double)p), 0.0);
}

// A wave's 1024 columns of one step from c on (a lane takes every 64th four, so that a load is
// contiguous); zeros past the row's last whole four.
struct Run {
  Quad a[kRun / 4], b[kRun / 4];
  __device__ __forceinline__ void load(const float* p, const float* q, int64_t c, int64_t vocab) {
    const int lane = threadIdx.x & 63;
    if (c + 64 * kRun <= vocab) {
#pragma unroll
      for (int i = 0; i < kRun / 4; ++i) {
        a[i] = *(const Quad*)(p + c + 256 * i + 4 * lane);
        b[i] = *(const Quad*)(q + c + 256 * i + 4 * lane);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kRun / 4; ++i) {
      const int64_t at = c + 256 * i + 4 * lane;
      a[i] = b[i] = Quad{{0.f, 0.f, 0.f, 0.f}};
      if (at + 4 <= vocab) {
        a[i] = *(const Quad*)(p + at);
        b[i] = *(const Quad*)(q + at);
      }
    }
  }
  // (LOOK: `odd` becomes NaN where a column is no number)
  template <bool LOOK>
  __device__ __forceinline__ double weight(float c_hi, float c_lo, float& odd) const {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kRun / 4; ++i) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (0 x is NaN for NaN and infinities: no distribution)
        if (LOOK) odd = __builtin_fmaf(0.f, a[i].v[e], __builtin_fmaf(0.f, b[i].v[e], odd));
        y[e] = fmaxf(__builtin_fmaf(-c_lo, b[i].v[e], __builtin_fmaf(-c_hi, b[i].v[e], a[i].v[e])), 0.f);
      }
      sum += (double)((y[0] + y[1]) + (y[2] + y[3]));
    }
    return sum;
  }
};

// Segment weights of a node's rows for C (0 with q = p: the target's own).  The first pass over a
// node (`fresh`) keeps its first steps in registers and in LDS, for the passes of the node's
// further rejections.
struct Held {
  Run step[kHeldSteps];
};
__device__ __forceinline__ void weigh(AcceptShared& sh, double* seg, Held& held, bool fresh, const float* p,
                                      const float* q, double C, int64_t vocab) {
  constexpr int kKept = kHeldSteps + kLdsSteps;
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int steps = (int)((vocab + kStep - 1) / kStep);
  const int64_t first = (int64_t)w * (64 * kRun);
  const float c_hi = (float)C, c_lo = (float)(C - (double)c_hi);
  float odd = 0.f;  // NaN where a column is
  auto close = [&](int step, double sum) {
    sum = wave_sum(sum);
    if (lane == 0) seg[step * kAccWaves + w] = sum;
  };
  auto kept = [&](int s) { return &sh.kept[s][0][0][t]; };
  if (fresh) {
#pragma unroll
    for (int s = 0; s < kHeldSteps; ++s) held.step[s].load(p, q, first + s * kStep, vocab);
  }
  // the first step that is streamed is on its way meanwhile
  Run cur, next;
  int step = fresh ? kHeldSteps : kKept;
  if (step < steps) cur.load(p, q, first + step * kStep, vocab);
  double sums[kHeldSteps] = {0.0, 0.0, 0.0, 0.0};
  if (fresh) {
#pragma unroll
    for (int s = 0; s < kHeldSteps; ++s)
      if (s < steps) sums[s] = held.step[s].weight<true>(c_hi, c_lo, odd);
  } else {
#pragma unroll
    for (int s = 0; s < kHeldSteps; ++s)
      if (s < steps) sums[s] = held.step[s].weight<false>(c_hi, c_lo, odd);
  }
  // (their exchanges side by side; steps past the row's are no segments)
#pragma unroll
  for (int s = 0; s < kHeldSteps; ++s) close(s, sums[s]);
  if (!fresh) {
#pragma unroll 1
    for (int s = kHeldSteps; s < min(steps, kKept); ++s) {
      const float4* const from = kept(s - kHeldSteps);
#pragma unroll
      for (int i = 0; i < kRun / 4; ++i) {
        const float4 a = from[i * kAccThreads], b = from[(kRun / 4 + i) * kAccThreads];
        next.a[i] = Quad{{a.x, a.y, a.z, a.w}};
        next.b[i] = Quad{{b.x, b.y, b.z, b.w}};
      }
      close(s, next.weight<false>(c_hi, c_lo, odd));
    }
  }
#pragma unroll 1
  for (; step < steps; ++step) {
    if (step + 1 < steps) next.load(p, q, first + (step + 1) * kStep, vocab);
    if (fresh && step < kKept) {
      float4* const to = kept(step - kHeldSteps);
#pragma unroll
      for (int i = 0; i < kRun / 4; ++i) {
        const Quad &a = cur.a[i], &b = cur.b[i];
        to[i * kAccThreads] = make_float4(a.v[0], a.v[1], a.v[2], a.v[3]);
        to[(kRun / 4 + i) * kAccThreads] = make_float4(b.v[0], b.v[1], b.v[2], b.v[3]);
      }
    }
    close(step, cur.weight<true>(c_hi, c_lo, odd));
    cur = next;
  }
  // the row's last columns, fewer than four, belong to the segment that they end
  const int64_t rest = vocab & ~(int64_t)3;
  if (rest < vocab && (rest / (64 * kRun)) % kAccWaves == w && lane == 0) {
    double sum = 0.0;
    for (int64_t at = rest; at < vocab; ++at) {
      odd += (p[at] - p[at]) + (q[at] - q[at]);
      sum += left_of(p[at], q[at], C);
    }
    seg[rest / (64 * kRun)] += sum;
  }
  if (__builtin_amdgcn_ballot_w64(odd != 0.f) != 0 && lane == 0)
    seg[w] = __longlong_as_double(0x7ff8000000000000ll);
  __syncthreads();
}

__device__ __forceinline__ double wave_incl(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o, RLT_WAVE);
    if (lane >= o) x += y;
  }
  return x;
}

// The total of a lane's run of segments, and of all (every wave alike).
__device__ __forceinline__ double lane_segments(const double* seg, int segments) {
  const int lane = threadIdx.x & 63, per = (segments + 63) / 64;
  double mine = 0.0;
  for (int i = 0; i < per; ++i)
    if (lane * per + i < segments) mine += seg[lane * per + i];
  return mine;
}

// The first column whose running weight passes `target` (one wave).
__device__ __forceinline__ int64_t draw(const double* weights, const float* p, const float* q, double C,
                                        int64_t vocab, int segments, double before, double target) {
  const int lane = threadIdx.x & 63, per = (segments + 63) / 64;
  // the last segment with weight at or before the target's: rounding may leave the running
  // weight's end short of it
  int seg = -1;
  double at = 0.0, run = before;
  for (int i = 0; i < per; ++i) {
    const int s = lane * per + i;
    if (s >= segments) break;
    if (weights[s] > 0.0 && run <= target) {
      seg = s;
      at = run;
    }
    run += weights[s];
  }
  const uint64_t has = __builtin_amdgcn_ballot_w64(seg >= 0);
  if (!has) return 0;
  const int owner = 63 - __builtin_clzll(has);
  seg = __shfl(seg, owner, RLT_WAVE);
  at = __shfl(at, owner, RLT_WAVE);
  const int64_t c = (int64_t)(seg / kAccWaves) * kStep + (int64_t)(seg % kAccWaves) * 64 * kRun + lane * kRun;
  // (here a lane's columns are consecutive)
  Quad a[kRun / 4], b[kRun / 4];
#pragma unroll
  for (int i = 0; i < kRun / 4; ++i) {
    const int64_t from = c + 4 * i;
    a[i] = b[i] = Quad{{0.f, 0.f, 0.f, 0.f}};
    if (from + 4 <= vocab) {
      a[i] = *(const Quad*)(p + from);
      b[i] = *(const Quad*)(q + from);
    } else {
      for (int e = 0; e < 3; ++e)
        if (from + e < vocab) {
          a[i].v[e] = p[from + e];
          b[i].v[e] = q[from + e];
        }
    }
  }
  double y[kRun], mine = 0.0;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    y[i] = left_of(a[i / 4].v[i % 4], b[i / 4].v[i % 4], C);
    mine += y[i];
  }
  const double incl = wave_incl(mine);
  double lane_before = __shfl_up(incl, 1, RLT_WAVE);
  if (lane == 0) lane_before = 0.0;
  run = at + lane_before;
  int col = -1;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    if (y[i] > 0.0 && run <= target) col = i;
    run += y[i];
  }
  const uint64_t lanes = __builtin_amdgcn_ballot_w64(col >= 0);
  if (!lanes) return 0;
  const int who = 63 - __builtin_clzll(lanes);
  return __shfl(c + col, who, RLT_WAVE);
}

__global__ __launch_bounds__(kAccThreads) void rlt_tree_accept_kernel(
    const int64_t* draft_tokens, const int64_t* parents, const int64_t* drafts, const float* q_all,
    const float* p_all, const float* u_accept, const float* u_final, int width, int64_t vocab,
    int64_t* path, int64_t* tokens, int64_t* accepted, int64_t* final_token, uint8_t* error) {
  __shared__ AcceptShared sh;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, nodes = width + 1;
  const float* const p = p_all + r * nodes * vocab;
  const float* const q = q_all + r * width * vocab;
  const int64_t d = drafts[r];
  const int live = (int)(d < 0 ? 0 : d > width ? width : d);
  bool bad = d != live;
  const float last_u = u_final[r];
  // every draft's two probabilities at its parent, in one round of loads
  for (int j = t; j < live; j += kAccThreads) {
    const int64_t parent = parents[r * width + j], token = draft_tokens[r * width + j];
    const bool child = parent >= 0 && parent <= j;
    sh.u[j] = u_accept[r * width + j];
    sh.parent[j] = child ? (int32_t)parent : -1;
    sh.token[j] = token;
    const bool in = child && token >= 0 && token < vocab;
    sh.px[j] = in ? p[parent * vocab + token] : 0.f;
    sh.qx[j] = in ? q[parent * vocab + token] : 0.f;  // 0: cannot have been drawn
  }
  if (t == 0) {
    sh.walk[0] = 0;
    sh.last = 0;
  }
  __syncthreads();
  const int segments = (int)((vocab + kStep - 1) / kStep) * kAccWaves;
  int node = 0, count = 0;
  double C = 0.0, R = 1.0;
  Held held;
  double* seg = sh.seg[1];
  // every wave walks alike: a lane holds the parents of drafts lane, lane + 64, ..
  int parent[(kMaxDrafts + 63) / 64];
#pragma unroll
  for (int k = 0; k < (kMaxDrafts + 63) / 64; ++k)
    parent[k] = lane + 64 * k < live ? sh.parent[lane + 64 * k] : -1;
  bool last = false;  // the pass over p alone, behind the walk
  for (int j = 0; !bad && !last;) {
    int child = live;
#pragma unroll
    for (int k = (kMaxDrafts + 63) / 64 - 1; k >= 0; --k) {
      const uint64_t b = __builtin_amdgcn_ballot_w64(lane + 64 * k >= j && parent[k] == node);
      if (b) child = 64 * k + __builtin_ctzll(b);
    }
    j = child;
    if (j < live) {
      const double px = sh.px[j], qx = sh.qx[j], u = sh.u[j];
      ++j;
      if (!(qx > 0.0) || !(fabs(px) < INFINITY) || !(qx < INFINITY)) {
        bad = true;
        break;
      }
      if (u * R * qx < __builtin_fma(-C, qx, px)) {
        ++count;
        node = j;
        if (t == 0) sh.walk[count] = node;
        C = 0.0;
        R = 1.0;
        continue;
      }
    } else if (C == 0.0) {
      last = true;
    } else {
      break;
    }
    const int64_t row = (int64_t)__builtin_amdgcn_readfirstlane(node) * vocab;
    const bool fresh = __builtin_amdgcn_readfirstlane(C == 0.0), alone = __builtin_amdgcn_readfirstlane(last);
    if (!last) C = two_floats(C + R);
    seg = seg == sh.seg[0] ? sh.seg[1] : sh.seg[0];  // (the last pass's may still be read)
    weigh(sh, seg, held, fresh, p + row, (alone ? p : q) + row, C, vocab);
    if (last) break;
    R = wave_sum(lane_segments(seg, segments));
    bad = !(R > 0.0) || !(R < INFINITY);
  }
  if (!bad) {
    if (t < 64) {
      const double incl = wave_incl(lane_segments(seg, segments)), total = __shfl(incl, 63, RLT_WAVE);
      double before = __shfl_up(incl, 1, RLT_WAVE);  // each lane's run
      if (lane == 0) before = 0.0;
      bad = !(total > 0.0) || !(total < INFINITY);
      if (!bad) {
        const double u = (double)last_u * total;
        // the draw stays below the total
        const double top = __longlong_as_double(__double_as_longlong(total) - 1);
        const float* const row = p + (int64_t)node * vocab;
        const int64_t token = draw(seg, row, C == 0.0 ? row : q + (int64_t)node * vocab, C, vocab, segments,
                                   before, u < top ? u : top);
        if (t == 0) sh.last = token;
      }
    }
  }
  if (t == 0) {
    accepted[r] = count;
    error[r] = bad ? 1 : 0;  // (thread 0 is in the drawing wave)
  }
  __syncthreads();
  if (t == 0) final_token[r] = sh.last;
  for (int i = t; i < nodes; i += kAccThreads) {
    path[r * nodes + i] = i <= count ? sh.walk[i] : -1;
    tokens[r * nodes + i] = i < count ? sh.token[sh.walk[i + 1] - 1] : i == count ? sh.last : 0;
  }
}

int64_t argmax_slices(int64_t vocab) {
  return (vocab + kSliceEpt * kThreads - 1) / (kSliceEpt * kThreads);
}

}  // namespace

extern "C" {

int rlt_tree_accept(const int64_t* draft_tokens, const int64_t* parents, const int64_t* drafts,
                    const float* q, const float* p, const float* u_accept, const float* u_final,
                    int64_t n, int32_t width, int64_t vocab, int64_t* path, int64_t* tokens,
                    int64_t* accepted, int64_t* final_token, uint8_t* error, hipStream_t stream) {
  if (n < 0 || width < 0 || vocab < 1) return RLT_ERR_ARGUMENT;
  if (width > kMaxDrafts || vocab > kMaxVocab || n >= kMaxRequests) return RLT_ERR_UNSUPPORTED;
  if (n == 0) return RLT_OK;
  if (!drafts || !p || !u_final || !path || !tokens || !accepted || !final_token || !error ||
      (width && (!draft_tokens || !parents || !q || !u_accept)))
    return RLT_ERR_ARGUMENT;
  hipLaunchKernelGGL(rlt_tree_accept_kernel, dim3((unsigned)n), dim3(kAccThreads), 0, stream,
                     draft_tokens, parents, drafts, q, p, u_accept, u_final, width, vocab, path,
                     tokens, accepted, final_token, error);
  return rlt_launch_status();
}

size_t rlt_greedy_tree_accept_workspace_size(int64_t n, int32_t width, int64_t vocab) {
  if (n <= 0 || width < 0 || width > kMaxDrafts || vocab < 1 || vocab > kMaxVocab) return 0;
  return (size_t)(n * (width + 1) * argmax_slices(vocab)) * sizeof(unsigned long long);
}

int rlt_greedy_tree_accept(const int64_t* draft_tokens, const int64_t* parents,
                           const int64_t* drafts, const void* target_logits, int32_t logits_dtype,
                           int64_t row_stride, int64_t n, int32_t width, int64_t vocab,
                           int64_t* targets, int64_t* path, int64_t* accepted, int64_t* next_token,
                           void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (n < 0 || width < 0 || vocab < 1) return RLT_ERR_ARGUMENT;
  if (n > 0 && n * (width + 1) > 1 && row_stride < vocab) return RLT_ERR_ARGUMENT;
  if (width > kMaxDrafts || vocab > kMaxVocab) return RLT_ERR_UNSUPPORTED;
  if (logits_dtype != RLT_F32 && logits_dtype != RLT_BF16 && logits_dtype != RLT_F16)
    return RLT_ERR_UNSUPPORTED;
  if (n == 0) return RLT_OK;
  const int64_t slices = argmax_slices(vocab), wgs = n * (width + 1) * slices;
  if (n > 0x7fffffff || wgs > kMaxLaunch / kThreads) return RLT_ERR_UNSUPPORTED;
  if (!drafts || !target_logits || !targets || !path || !accepted || !next_token ||
      (width && (!draft_tokens || !parents)))
    return RLT_ERR_ARGUMENT;
  if (!workspace || (uintptr_t)workspace % 8 ||
      workspace_bytes < rlt_greedy_tree_accept_workspace_size(n, width, vocab))
    return RLT_ERR_WORKSPACE;
  unsigned long long* const best = (unsigned long long*)workspace;
#define RLT_TREE_ARGMAX(DT)                                                                     \
  hipLaunchKernelGGL((rlt_tree_argmax_kernel<DT>), dim3((unsigned)wgs), dim3(kThreads), 0, stream, \
                     target_logits, row_stride, vocab, (int)slices, best)
  switch (logits_dtype) {
    case RLT_F32: RLT_TREE_ARGMAX(RLT_F32); break;
    case RLT_BF16: RLT_TREE_ARGMAX(RLT_BF16); break;
    default: RLT_TREE_ARGMAX(RLT_F16); break;
  }
#undef RLT_TREE_ARGMAX
  hipLaunchKernelGGL(rlt_greedy_tree_kernel, dim3((unsigned)n), dim3(kThreads), 0, stream, best,
                     (int)slices, draft_tokens, parents, drafts, width, targets, path, accepted,
                     next_token);
  return rlt_launch_status();
}

}  // extern "C"
