// Speculative decoding around the attention: the rows of trees of drafted tokens (what a row sees, its position, its place in the cache), verification of the
// drafted tokens against the target's logits, and the move of the accepted rows' keys and values to the places that they keep.
//
// The rows of all sequences' trees lie one after the other, sequence b's from cu[b] to cu[b + 1]; row 0 is the last token that is decided, row j continues
// row parents[j] < j of its sequence. Row j's key and value stand at place ctx[b] + j of the sequence's pages.
//
// This file is compiled without fast math.
#include "common.cuh"

#include <math.h>

namespace {
using namespace rlb;

constexpr int DR_ROWS = 256;      // rows of a tree

struct TreeSpan {
  int lo, n;
};
// Rows of sequence b; offsets that do not ascend within [0, T], or more rows than the caller counts with, are reported and cut.
__device__ __forceinline__ TreeSpan tree_span(const int* cu, int b, int T, int max_rows, int* status, bool report) {
  const int a = cu[b], e = cu[b + 1];
  const int lo = min(max(a, 0), T), hi = min(max(e, lo), T);
  const int n = min(hi - lo, max_rows);
  if (report && (lo != a || lo + n != e) && status) atomicCAS(status, 0, RLB_ERR_BOUNDS);
  return {lo, n};
}

// ------------------------------------------------------------------------------------------------ rows
// One CTA per sequence (and one for the rows behind the last), a thread per row: it walks up its parents.
__global__ void __launch_bounds__(DR_ROWS)
tree_rows_kernel(const int* __restrict__ parents, const int* __restrict__ cu, const int* __restrict__ ctx, const int* __restrict__ table, long long table_ld,
                 int pages, int block, int B, int T, int max_rows, int words, int* __restrict__ masks, int* __restrict__ positions,
                 long long* __restrict__ slots, int* status) {
  __shared__ int up[DR_ROWS];
  pdl_sync();
  const int b = blockIdx.x, j = threadIdx.x;
  if (b == B) {      // rows of no sequence see nothing and have no place
    const int end = B > 0 ? min(max(cu[B], 0), T) : 0;
    for (long long t = end + j; t < T; t += blockDim.x) {
      for (int w = 0; w < words; ++w) masks[t * words + w] = 0;
      positions[t] = 0;
      slots[t] = -1;
    }
    return;
  }
  const TreeSpan s = tree_span(cu, b, T, max_rows, status, j == 0);
  if (j < s.n) {
    const int p = parents[s.lo + j];
    up[j] = p >= 0 && p < j ? p : -1;
    if ((p >= j || p < -1) && status) atomicCAS(status, 0, RLB_ERR_BOUNDS);
  }
  __syncthreads();
  if (j >= s.n) return;
  uint32_t bits[DR_ROWS / 32] = {};
  int depth = 0;
  for (int a = j; a >= 0; a = up[a], ++depth) {
#pragma unroll
    for (int w = 0; w < DR_ROWS / 32; ++w) bits[w] |= a >> 5 == w ? 1u << (a & 31) : 0u;
  }
  const long long t = s.lo + j;
#pragma unroll
  for (int w = 0; w < DR_ROWS / 32; ++w)
    if (w < words) masks[t * words + w] = static_cast<int>(bits[w]);
  positions[t] = ctx[b] + depth - 1;
  const long long place = static_cast<long long>(ctx[b]) + j, page = place / block;
  const bool in = place >= 0 && page < pages;
  if (!in && status) atomicCAS(status, 0, RLB_ERR_BOUNDS);
  slots[t] = in ? static_cast<long long>(table[b * table_ld + page]) * block + place % block : -1;
}

// ------------------------------------------------------------------------------------------------ keep
constexpr int KEEP_PAIRS = 60;
struct KeepCaches {
  uint4* p[2 * KEEP_PAIRS];
};
// One CTA per tensor and sequence: each thread has 16 bytes of a head and moves them row by row in ascending order, four rows loaded before they are stored (a row's
// source lies behind the targets of all rows before it).
__global__ void __launch_bounds__(256)
keep_kernel(const __grid_constant__ KeepCaches caches, const int* __restrict__ table, long long table_ld, int pages, int block, int blocks, int heads, int vecs,
            const int* __restrict__ ctx, const int* __restrict__ rows, int S, const int* __restrict__ counts, int* status) {
  pdl_sync();
  const int b = blockIdx.y;
  uint4* c = caches.p[blockIdx.x];
  const int n = min(counts[b], S);
  const long long first = ctx[b];
  const long long at = static_cast<long long>(b) * S;
  auto place = [&](long long q) -> long long {      // 16-byte words before this place's of head 0, -1 where there is none
    const long long page = q / block;
    if (q < 0 || page >= pages) return -1;
    const int id = table[b * table_ld + page];
    return id < 0 || id >= blocks ? -1 : (static_cast<long long>(id) * heads * block + q % block) * vecs;
  };
  for (int u = threadIdx.x; u < heads * vecs; u += blockDim.x) {
    const long long off = static_cast<long long>(u / vecs) * block * vecs + u % vecs;
    int last = -1;
    for (int i0 = 0; i0 < n; i0 += 4) {
      uint4 v[4];
      long long to[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + k;
        to[k] = -1;
        if (i >= n) continue;
        const int r = rows[at + i];
        const bool bad = r <= last || r < i;
        last = bad ? last : r;
        if (r == i) continue;
        const long long from = bad ? -1 : place(first + r), dst = place(first + i);
        if (from < 0 || dst < 0) {
          if (status) atomicCAS(status, 0, RLB_ERR_BOUNDS);
          continue;
        }
        to[k] = dst;
        v[k] = c[from + off];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (to[k] >= 0) c[to[k] + off] = v[k];
    }
  }
}

// ------------------------------------------------------------------------------------------------ verification
struct VerifyArgs {
  const void* logits;
  const void* draft;      // null: children are taken without chance
  long long ld, ld_draft;
  int V, T, max_rows, steps, greedy;
  const int* tokens;
  const int* parents;
  const int* cu;
  const float* uniforms;
  const float* temps;      // null: temp
  double temp;
  int* out_tokens;
  int* out_counts;
  int* out_rows;
  float* out_logprobs;
  int* status;
};

constexpr int DV_THREADS = 1024, DV_WARPS = DV_THREADS / 32;
constexpr double LOG2E = 1.4426950408889634074;

// NaN weighs nothing, +inf as much as the largest number.
__device__ __forceinline__ float usable(float x) { return x != x ? -INFINITY : fminf(x, 3.402823466e38f); }
__device__ __forceinline__ float logit(const float* p, int i) { return usable(p[i]); }
__device__ __forceinline__ float logit(const __nv_bfloat16* p, int i) { return usable(__bfloat162float(p[i])); }

struct Peak {
  float x;
  int at;
};
__device__ __forceinline__ Peak higher(Peak a, Peak b) { return b.x > a.x || (b.x == a.x && b.at < a.at) ? b : a; }
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One CTA per sequence, which walks down the accepted rows and reads the logits of the rows that it comes to. All in 64 bits.
template <typename T, bool DRAFT>
__global__ void __launch_bounds__(DV_THREADS)
verify_kernel(const VerifyArgs a) {
  __shared__ int up[DR_ROWS], tok[DR_ROWS], gone[DR_ROWS];
  __shared__ float num[DR_ROWS];
  __shared__ double left[DR_ROWS + 1];      // sums of what is left to be given after so many rejections
  __shared__ double part[DV_WARPS];
  __shared__ Peak peaks[DV_WARPS];
  __shared__ int found;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_sync();
  const TreeSpan s = tree_span(a.cu, b, a.T, a.max_rows, a.status, tid == 0);
  for (int i = tid; i < a.steps; i += DV_THREADS) {
    const long long o = static_cast<long long>(b) * a.steps + i;
    a.out_tokens[o] = -1;
    a.out_rows[o] = -1;
    a.out_logprobs[o] = 0.f;
  }
  if (s.n == 0) {
    if (tid == 0) a.out_counts[b] = 0;
    return;
  }
  for (int j = tid; j < s.n; j += DV_THREADS) {
    up[j] = j ? a.parents[s.lo + j] : -1;
    tok[j] = a.tokens[s.lo + j];
    num[j] = a.uniforms[s.lo + j];
  }
  const float given = a.temps ? a.temps[b] : static_cast<float>(a.temp);
  const bool greedy = a.greedy || !(given > 0.f);
  const double temp = !(given > 0.f) ? 1.0 : a.temps ? static_cast<double>(given) : a.temp, c = LOG2E / temp;
  const int share = ((a.V + DV_WARPS - 1) / DV_WARPS + 31) / 32 * 32, w0 = min(a.V, warp * share), w1 = min(a.V, w0 + share);      // a warp's columns

  auto total = [&](double v) {      // over the CTA, in the warps' order
    v = warp_sum_d(v);
    __syncthreads();
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = 0.0;
    for (int i = 0; i < DV_WARPS; ++i) v += part[i];
    return v;
  };
  auto peak = [&](const T* z) {
    Peak v{-INFINITY, 0x7fffffff};
    for (int i = w0 + lane; i < w1; i += 32) v = higher(v, Peak{logit(z, i), i});
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = higher(v, Peak{__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.at, o)});
    __syncthreads();
    if (lane == 0) peaks[warp] = v;
    __syncthreads();
    v = peaks[0];
    for (int i = 1; i < DV_WARPS; ++i) v = higher(v, peaks[i]);
    return v;
  };
  auto weight = [&](float x, float top) { return x == -INFINITY ? 0.0 : exp2((static_cast<double>(x) - static_cast<double>(top)) * c); };

  int node = 0, count = 0;
  __syncthreads();
  while (true) {
    const T* z = static_cast<const T*>(a.logits) + (s.lo + node) * a.ld;
    const T* d = DRAFT ? static_cast<const T*>(a.draft) + (s.lo + node) * a.ld_draft : nullptr;
    const Peak top = peak(z);
    double sum = 0.0;
    for (int i = w0 + lane; i < w1; i += 32) sum += weight(logit(z, i), top.x);
    sum = total(sum);
    float dtop = 0.f;
    double dsum = 1.0;
    if (DRAFT && !greedy) {
      dtop = peak(d).x;
      dsum = 0.0;
      for (int i = w0 + lane; i < w1; i += 32) dsum += weight(logit(d, i), dtop);
      dsum = total(dsum);
    }
    const bool some = top.x > -INFINITY;      // a row without a number above -inf has no probabilities
    int rejected = 0, next = -1;
    // what is left of token i's probability after `r` rejections
    auto rest = [&](int i, int r) {
      double w = some ? weight(logit(z, i), top.x) / sum : 0.0;
      if (DRAFT) {
        if (r > 0) {
          const double q = dtop > -INFINITY ? weight(logit(d, i), dtop) / dsum : 0.0;
          for (int k = 0; k < r; ++k) w = fmax(w / left[k] - q, 0.0);
        }
      } else {
        for (int k = 0; k < r; ++k) w = gone[k] == i ? 0.0 : w;
      }
      return w;
    };
    if (tid == 0) left[0] = 1.0;
    __syncthreads();
    for (int j = node + 1; j < s.n && next < 0 && count + 1 < a.steps; ++j) {
      if (up[j] != node) continue;
      const int t = tok[j];
      if (greedy) {
        if (some && t == top.at) next = j;
        continue;
      }
      if (t < 0 || t >= a.V) continue;      // has no probability, and is none of the draft's
      const double w = rest(t, rejected);
      const double q = DRAFT ? (dtop > -INFINITY ? weight(logit(d, t), dtop) / dsum : 0.0) : 1.0;
      if (static_cast<double>(num[j]) * q * left[rejected] < w) {
        next = j;
        break;
      }
      if (DRAFT) {
        ++rejected;
        double v = 0.0;
        for (int i = w0 + lane; i < w1; i += 32) v += rest(i, rejected);
        v = total(v);
        if (tid == 0) left[rejected] = v;
        __syncthreads();
        if (!(v > 0.0)) break;
      } else if (w > 0.0) {
        __syncthreads();
        if (tid == 0) {
          gone[rejected] = t;
          left[rejected + 1] = left[rejected] - w;
        }
        ++rejected;
        __syncthreads();
      }
    }
    int t = next >= 0 ? tok[next] : top.at;
    if (next < 0 && !some) t = 0;
    if (next < 0 && !greedy && some) {      // draw from what is left: the first token whose share of the running sum passes the number
      double mine = 0.0, all = 0.0;
      for (int again = 0; again < 2; ++again) {
        mine = 0.0;
        for (int i = w0 + lane; i < w1; i += 32) mine += rest(i, rejected);
        mine = warp_sum_d(mine);
        all = total(lane == 0 ? mine : 0.0);
        if (all > 0.0) break;
        rejected = 0;
      }
      double before = 0.0;
      for (int i = 0; i < warp; ++i) before += part[i];
      const double aim = static_cast<double>(num[0]) * all;
      if (tid == 0) found = 0x7fffffff;
      __syncthreads();
      if (lane == 0 && mine > 0.0 && before + mine > aim) atomicMin(&found, warp);
      __syncthreads();
      bool over_all = found == 0x7fffffff;      // a number of 1 and more, or none: the last token that has a share
      __syncthreads();
      if (over_all && lane == 0 && mine > 0.0) atomicMin(&found, DV_WARPS - 1 - warp);
      __syncthreads();
      if (warp == (over_all ? DV_WARPS - 1 - found : found)) {
        int last = 0, hit = -1;
        for (int i0 = w0; i0 < w1 && hit < 0; i0 += 32) {
          const int i = i0 + lane;
          const double w = i < w1 ? rest(i, rejected) : 0.0;
          double run = w;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
          }
          const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && before + run > aim), any = __ballot_sync(0xffffffffu, w > 0.0);
          if (over) hit = i0 + __ffs(over) - 1;
          if (any) last = i0 + 31 - __clz(any);
          before += __shfl_sync(0xffffffffu, run, 31);
        }
        if (lane == 0) peaks[0].at = hit >= 0 ? hit : last;
      }
      __syncthreads();
      t = peaks[0].at;
      __syncthreads();
    }
    if (tid == 0) {
      const long long o = static_cast<long long>(b) * a.steps + count;
      a.out_rows[o] = node;
      a.out_tokens[o] = t;
      a.out_logprobs[o] = !some ? -INFINITY : static_cast<float>((static_cast<double>(logit(z, t)) - static_cast<double>(top.x)) / temp - log(sum));
    }
    ++count;
    if (next < 0) break;
    node = next;
  }
  if (tid == 0) a.out_counts[b] = count;
}
}  // namespace

RLB_API int rlb_tree_rows(const int* parents, const int* cu, const int* ctx, const int* table, long long table_ld, int pages, int block, int B, int T, int max_rows,
                          int words, int* masks, int* positions, long long* slots, int* status, void* stream) {
  if (B < 0 || T < 0 || max_rows < 1 || max_rows > DR_ROWS || words * 32 < max_rows || block < 1) return -2;
  return static_cast<int>(rlb_launch_pdl(tree_rows_kernel, dim3(B + 1), dim3(DR_ROWS), 0, static_cast<cudaStream_t>(stream), parents, cu, ctx, table, table_ld, pages, block,
                                         B, T, max_rows, words, masks, positions, slots, status));
}

// caches: `tensors` pointers (host) to caches of the same shape [blocks, heads, block, vecs 16-byte words].
RLB_API int rlb_kv_keep(void* const* caches, int tensors, const int* table, long long table_ld, int pages, int block, int blocks, int heads, int vecs, const int* ctx,
                        const int* rows, int S, const int* counts, int B, int* status, void* stream) {
  if (B > 65535 || block < 1) return -2;
  for (int t0 = 0; t0 < tensors; t0 += 2 * KEEP_PAIRS) {
    KeepCaches c;
    const int n = tensors - t0 < 2 * KEEP_PAIRS ? tensors - t0 : 2 * KEEP_PAIRS;
    for (int i = 0; i < n; ++i) c.p[i] = static_cast<uint4*>(caches[t0 + i]);
    for (int i = n; i < 2 * KEEP_PAIRS; ++i) c.p[i] = nullptr;
    const cudaError_t e = rlb_launch_pdl(keep_kernel, dim3(n, B), dim3(256), 0, static_cast<cudaStream_t>(stream), c, table, table_ld, pages, block, blocks, heads, vecs,
                                         ctx, rows, S, counts, status);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return 0;
}

RLB_API int rlb_verify_drafts(const void* logits, long long ld, const void* draft, long long ld_draft, int f32, int V, int T, int B, int max_rows, int steps,
                              const int* tokens, const int* parents, const int* cu, const float* uniforms, const float* temps, double temp, int greedy,
                              int* out_tokens, int* out_counts, int* out_rows, float* out_logprobs, int* status, void* stream) {
  if (max_rows < 1 || max_rows > DR_ROWS || steps < 1 || steps > max_rows || V < 1) return -2;
  const VerifyArgs a{logits, draft, ld, ld_draft, V, T, max_rows, steps, greedy, tokens, parents, cu, uniforms, temps, temp, out_tokens, out_counts, out_rows,
                     out_logprobs, status};
  auto k = f32 ? (draft ? verify_kernel<float, true> : verify_kernel<float, false>)
               : (draft ? verify_kernel<__nv_bfloat16, true> : verify_kernel<__nv_bfloat16, false>);
  return static_cast<int>(rlb_launch_pdl(k, dim3(B), dim3(DV_THREADS), 0, static_cast<cudaStream_t>(stream), a));
}
