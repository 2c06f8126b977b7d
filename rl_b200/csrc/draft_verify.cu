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
// p = softmax(l / T) of a node, in 64 bits throughout: the last token is the first whose running sum passes a given number, and with 32 bits the running sums of a flat
// distribution over 10^5 tokens would be off by as much as a token has. A weight is e = 2^((l - m) log2(e) / T), taken as 2^(k / 256) from a table times a polynomial of third degree
// in the rest r, |r| <= 1 / 512, whose error is (r ln 2)^4 / 24 < 1.5e-13: ten instructions of the 64-bit pipe, which has half the rate of the 32-bit one.
//
// A cluster of CTAs has a sequence. It walks down the accepted rows and reads the logits of these rows alone, which is what the operator cannot do without: each warp has a range
// of tokens and leaves its sum in every CTA's shared memory; all CTAs come to the same decision. The ranges' sums say in which range the last token lies, whose warp
// goes through it once more. Where tokens have been rejected the sums are taken again first: with draft logits all of them, otherwise the ranges that a rejected token was in.
//
// Bound by the 64-bit pipe and, for few sequences, by latency: the row, the exchange and the decision one after another.
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

constexpr int DV_THREADS = 512, DV_WARPS = DV_THREADS / 32, DV_CLUSTER = 8, DV_PARTS = DV_WARPS * DV_CLUSTER;
constexpr int EXP_STEPS = 256;
constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.69314718055994530942;
constexpr float F_MAX = 3.402823466e38f;

// NaN weighs nothing, +inf as much as the largest number.
__device__ __forceinline__ float usable(float x) { return fminf(fmaxf(x, -INFINITY), F_MAX); }
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Weights relative to the logit m. Logits below `low` weigh nothing (2^-1000 of m's), those above `high` would pass 2^800.
struct Scale {
  double m;
  float low, high;
  // octave: the difference of logits that doubles a weight
  __device__ __forceinline__ void set(float top, double octave) {
    m = static_cast<double>(top);
    low = fmaxf(fminf(__double2float_ru(m - 1000.0 * octave), top), -F_MAX);
    high = fmaxf(__double2float_rd(m + 800.0 * octave), top);
  }
  __device__ __forceinline__ double operator()(const double* table, double c, float x) const {
    const double z = (static_cast<double>(x) - m) * c;
    const double magic = 6755399441055744.0 / EXP_STEPS;      // 1.5 * 2^52 / 256: the sum's low word is the nearest number of 256ths
    const double t = z + magic, r = z - (t - magic);
    const int k = __double2loint(t);
    const double p = r * (LN2 + r * (LN2 * LN2 / 2 + r * (LN2 * LN2 * LN2 / 6)));
    const double f = table[k & (EXP_STEPS - 1)];
    const bool none = !(x >= low);
    const double s = __hiloint2double(none ? 0 : __double2hiint(f) + (k >> 8 << 20), none ? 0 : __double2loint(f));
    return none ? 0.0 : fma(s, p, s);
  }
};

__device__ __forceinline__ void push_d(uint32_t addr, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory"); }

struct Part {      // of a warp's range
  double m, sum;      // sum of weights relative to m (-inf: none)
  double dm, dsum;    // of the draft's
  float peak;
  int at;
};

template <typename T, int ELEMS>      // logits a lane has at a time
struct RowLogits {
  static constexpr int VEC = 16 / sizeof(T), LOADS = ELEMS / VEC;
  const T* p;
  int V;
  int shift;      // elements before the row's first that its first group of 16 bytes has
  bool vec;
  // group g: elements g * VEC - shift and on; those outside of the row are -inf
  __device__ __forceinline__ uint4 load(int g, int g1) const {
    const int e = g * VEC - shift;
    uint4 v;
    uint32_t* w = &v.x;
    if (g < g1 && vec && e >= 0 && e + VEC <= V) return __ldg(reinterpret_cast<const uint4*>(p + e));
    if (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = g < g1 && e + i >= 0 && e + i < V ? reinterpret_cast<const uint32_t*>(p)[e + i] : 0xff800000u;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int a = e + 2 * i;
        const uint32_t lo = g < g1 && a >= 0 && a < V ? reinterpret_cast<const uint16_t*>(p)[a] : 0xff80u;
        const uint32_t hi = g < g1 && a + 1 >= 0 && a + 1 < V ? reinterpret_cast<const uint16_t*>(p)[a + 1] : 0xff80u;
        w[i] = lo | hi << 16;
      }
    }
    return v;
  }
  static __device__ __forceinline__ float element(const uint4& v, int i) {
    const uint32_t* w = &v.x;
    return usable(sizeof(T) == 4 ? __uint_as_float(w[i]) : __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16));
  }
  __device__ __forceinline__ float at(int i) const { return usable(static_cast<float>(p[i])); }
};

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(DV_THREADS, 2)
verify_kernel(const VerifyArgs a) {
  using Row = RowLogits<T, DRAFT ? 8 : 16>;
  constexpr int VEC = Row::VEC, LOADS = Row::LOADS;
  __shared__ double table[EXP_STEPS];
  __shared__ Part parts[2][DV_PARTS];      // of all warps of the cluster, by turns
  __shared__ int up[DR_ROWS], tok[DR_ROWS], gone[DR_ROWS];
  __shared__ float num[DR_ROWS], lz[DR_ROWS], ld[DR_ROWS];      // numbers, logits of the children's tokens in their parent's rows
  __shared__ double left[DR_ROWS + 1];                          // what is left to be given after so many rejections
  __shared__ int verdict, tried, turned_down;
  __shared__ double share[DV_PARTS];      // the ranges' probabilities
  __shared__ double row_top, row_sum, row_inv, draft_top, draft_inv;
  __shared__ int row_best;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int rank = static_cast<int>(cluster_ctarank()), b = blockIdx.x / ctas, W = static_cast<int>(ctas) * DV_WARPS, me = rank * DV_WARPS + warp;
  if (tid < EXP_STEPS) table[tid] = exp2(static_cast<double>(tid) / EXP_STEPS);
  pdl_sync();
  const TreeSpan s = tree_span(a.cu, b, a.T, a.max_rows, a.status, tid == 0 && rank == 0);
  const long long out = static_cast<long long>(b) * a.steps;
  int count = 0;
  if (s.n > 0) {
    for (int j = tid; j < s.n; j += DV_THREADS) {
      up[j] = j ? a.parents[s.lo + j] : -1;
      tok[j] = a.tokens[s.lo + j];
      num[j] = a.uniforms[s.lo + j];
    }
    const float given = a.temps ? a.temps[b] : static_cast<float>(a.temp);
    const bool cold = a.greedy || !(given > 0.f);
    const double temp = !(given > 0.f) ? 1.0 : a.temps ? static_cast<double>(given) : a.temp, c = LOG2E / temp, octave = 1.0 / c;
    int turn = 0;
    cluster_arrive();      // (all CTAs of the cluster run before one writes into another's memory)
    cluster_wait();

    auto exchange = [&](double m, double sum, double dm, double dsum, float peak, int at) {      // this warp's part to all CTAs
      turn ^= 1;
      if (lane < static_cast<int>(ctas)) {
        Part* p = &parts[turn][me];
        push_d(mapa_shared(smem_u32(&p->m), lane), m);
        push_d(mapa_shared(smem_u32(&p->sum), lane), sum);
        if (DRAFT) {
          push_d(mapa_shared(smem_u32(&p->dm), lane), dm);
          push_d(mapa_shared(smem_u32(&p->dsum), lane), dsum);
        }
        push_d(mapa_shared(smem_u32(&p->peak), lane), __hiloint2double(at, __float_as_int(peak)));
      }
      cluster_arrive();
      cluster_wait();
    };

    int node = 0;
    while (true) {
      Row z{static_cast<const T*>(a.logits) + (s.lo + node) * a.ld, a.V, 0, true}, d{};
      z.shift = static_cast<int>(reinterpret_cast<uintptr_t>(z.p) % 16 / sizeof(T));
      if (DRAFT) {
        d = Row{static_cast<const T*>(a.draft) + (s.lo + node) * a.ld_draft, a.V, z.shift, false};
        d.vec = reinterpret_cast<uintptr_t>(d.p) % 16 / sizeof(T) == z.shift;
      }
      const int groups = (a.V + z.shift + VEC - 1) / VEC, per = (groups + W - 1) / W, g0 = min(groups, me * per), g1 = min(groups, g0 + per);
      for (int j = tid; j < s.n; j += DV_THREADS)
        if (j > node && up[j] == node && tok[j] >= 0 && tok[j] < a.V) {
          lz[j] = z.at(tok[j]);
          if (DRAFT) ld[j] = d.at(tok[j]);
        }
      // the range's groups, LOADS of them a lane at a time, the next ones on their way
      auto each = [&](auto&& fn) {
        uint4 vz[LOADS], vd[DRAFT ? LOADS : 1];
        auto fetch = [&](int g) {
#pragma unroll
          for (int u = 0; u < LOADS; ++u) {
            vz[u] = z.load(g + u * 32 + lane, g1);
            if (DRAFT) vd[u] = d.load(g + u * 32 + lane, g1);
          }
        };
        fetch(g0);
        for (int g = g0; g < g1; g += 32 * LOADS) {
          uint4 wz[LOADS], wd[DRAFT ? LOADS : 1];
#pragma unroll
          for (int u = 0; u < LOADS; ++u) {
            wz[u] = vz[u];
            if (DRAFT) wd[u] = vd[u];
          }
          if (g + 32 * LOADS < g1) fetch(g + 32 * LOADS);
          if (!fn(g, wz, wd)) break;
        }
      };
      // ---------------------------------------------------------------- the sums of the row
      float peak = -INFINITY;
      int at = 0x7fffffff;
      double sum = 0.0, dsum = 0.0;
      Scale sc, dsc;
      sc.m = dsc.m = -INFINITY;
      sc.high = dsc.high = -INFINITY;
      auto add = [&](Scale& q, double& total, const uint4 (&v)[LOADS]) {
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < LOADS; ++u)
#pragma unroll
          for (int i = 0; i < VEC; ++i) top = fmaxf(top, Row::element(v[u], i));
        if (__any_sync(0xffffffffu, top > q.high)) {      // the first numbers, or far larger ones
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const double before = q.m;
          q.set(top, octave);
          total = before == -INFINITY ? 0.0 : total * exp2((before - q.m) * c);
        }
        if (q.m == -INFINITY) return;
#pragma unroll
        for (int u = 0; u < LOADS; ++u)
#pragma unroll
          for (int i = 0; i < VEC; ++i) total += q(table, c, Row::element(v[u], i));
      };
      each([&](int g, const uint4 (&wz)[LOADS], const uint4 (&wd)[DRAFT ? LOADS : 1]) {
        add(sc, sum, wz);
        if (DRAFT) {
          if (!cold) add(dsc, dsum, reinterpret_cast<const uint4(&)[LOADS]>(wd));
        }
        if (cold) {
#pragma unroll
          for (int u = 0; u < LOADS; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float x = Row::element(wz[u], i);
              if (x > peak) {
                peak = x;
                at = (g + u * 32 + lane) * VEC - z.shift + i;
              }
            }
        }
        return true;
      });
      sum = warp_sum_d(sum);
      if (DRAFT) dsum = warp_sum_d(dsum);
      if (cold) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const float x = __shfl_xor_sync(0xffffffffu, peak, o);
          const int i = __shfl_xor_sync(0xffffffffu, at, o);
          if (x > peak || (x == peak && i < at)) {
            peak = x;
            at = i;
          }
        }
      }
      exchange(sc.m, sum, dsc.m, dsum, peak, at);
      // the first warp joins the parts: lane i has four of them, in their order
      if (warp == 0) {
        const Part* got = parts[turn];
        double mine[4], top = -INFINITY, dtop = -INFINITY, all = 0.0, dall = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int w = lane * 4 + k;
          if (w >= W) continue;
          top = fmax(top, got[w].m);
          if (DRAFT) dtop = fmax(dtop, got[w].dm);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (DRAFT) dtop = fmax(dtop, __shfl_xor_sync(0xffffffffu, dtop, o));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int w = lane * 4 + k;
          mine[k] = w < W && got[w].m > -INFINITY ? got[w].sum * exp2((got[w].m - top) * c) : 0.0;
          all += mine[k];
          if (DRAFT) dall += w < W && got[w].dm > -INFINITY ? got[w].dsum * exp2((got[w].dm - dtop) * c) : 0.0;
        }
        all = warp_sum_d(all);
        if (DRAFT) dall = warp_sum_d(dall);
        const double inv = top > -INFINITY ? 1.0 / all : 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) share[lane * 4 + k] = mine[k] * inv;
        if (lane == 0) {
          row_top = top;
          row_sum = all;
          row_inv = inv;
          if (DRAFT) {
            draft_top = dtop;
            draft_inv = dtop > -INFINITY ? 1.0 / dall : 0.0;
          }
          int best = 0x7fffffff;
          if (cold) {
            float x = -INFINITY;
            for (int w = 0; w < W; ++w)
              if (got[w].peak > x) {      // (parts lie in the tokens' order)
                x = got[w].peak;
                best = got[w].at;
              }
          }
          row_best = best;
          left[0] = 1.0;
          tried = node;
          turned_down = 0;
        }
      }
      __syncthreads();
      const double top = row_top, inv = row_inv, dinv = DRAFT ? draft_inv : 0.0;
      const bool some = top > -INFINITY;      // a row without a number above -inf has no probabilities
      Scale p, q;      // of the whole row
      p.set(static_cast<float>(some ? top : 0.0), octave);
      if (DRAFT) q.set(static_cast<float>(dinv > 0.0 ? draft_top : 0.0), octave);
      // what is left of the probability of a token after `r` rejections, from its logits
      int rejected = 0;
      auto rest = [&](int i, float x, float y, int r) {
        double w = p(table, c, x) * inv;
        if (DRAFT) {
          if (r > 0) {
            const double g = q(table, c, y) * dinv;
            for (int k = 0; k < r; ++k) w = fmax(w / left[k] - g, 0.0);
          }
        } else {
          for (int k = 0; k < r; ++k) w = gone[k] == i ? 0.0 : w;
        }
        return w;
      };
      auto sum_rest = [&](int r) {      // over this warp's range
        double v = 0.0;
        each([&](int g, const uint4 (&wz)[LOADS], const uint4 (&wd)[DRAFT ? LOADS : 1]) {
#pragma unroll
          for (int u = 0; u < LOADS; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) v += rest((g + u * 32 + lane) * VEC - z.shift + i, Row::element(wz[u], i), DRAFT ? Row::element(wd[DRAFT ? u : 0], i) : 0.f, r);
          return true;
        });
        return warp_sum_d(v);
      };
      double mine[4], total = 0.0;
      auto take = [&](double v) {      // this warp's part of new sums; the parts and the whole sum of all
        exchange(0.0, v, 0.0, 0.0, 0.f, 0);
        total = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          mine[k] = lane * 4 + k < W ? parts[turn][lane * 4 + k].sum : 0.0;
          total += mine[k];
        }
        total = warp_sum_d(total);
      };
      // ---------------------------------------------------------------- the children
      int next = -1;
      while (true) {
        if (tid == 0) {      // verdict: an accepted row, -1 none, -2 one rejected after which the sums are taken again
          int v = -1, j = tried + 1, r = rejected;
          for (; j < s.n && v == -1 && count + 1 < a.steps; ++j) {
            if (up[j] != node) continue;
            const int t = tok[j];
            if (cold) {
              if (some && t == row_best) v = j;
              continue;
            }
            if (t < 0 || t >= a.V) continue;      // has no probability, and is none of the draft's
            const double w = rest(t, lz[j], DRAFT ? ld[j] : 0.f, r);
            const double g = DRAFT ? q(table, c, ld[j]) * dinv : 1.0;
            if (static_cast<double>(num[j]) * g * left[r] < w) {
              v = j;
            } else if (DRAFT) {
              v = -2;
            } else if (w > 0.0) {
              gone[r] = t;
              left[r + 1] = left[r] - w;
              ++r;
            }
          }
          tried = j - 1;
          verdict = v;
          if (!DRAFT) turned_down = r;
        }
        __syncthreads();
        const int v = verdict;
        if (!DRAFT) rejected = turned_down;
        if (v != -2) {
          next = v;
          break;
        }
        ++rejected;
        take(sum_rest(rejected));
        if (tid == 0) left[rejected] = total;
        __syncthreads();
        if (!(total > 0.0)) break;
      }
      // ---------------------------------------------------------------- the token
      const auto logprob = [&](float x) { return some ? static_cast<float>((static_cast<double>(x) - top) / temp - log(row_sum)) : -INFINITY; };
      if (rank == 0 && tid == 0) a.out_rows[out + count] = node;
      if (next >= 0) {
        if (rank == 0 && tid == 0) {
          a.out_tokens[out + count] = tok[next];
          a.out_logprobs[out + count] = logprob(lz[next]);
        }
        ++count;
        node = next;
        __syncthreads();      // (the rejections of this row have been read)
        continue;
      }
      if (cold || !some) {
        if (rank == 0 && tid == 0) {
          const int t = some ? row_best : 0;
          a.out_tokens[out + count] = t;
          a.out_logprobs[out + count] = logprob(some ? z.at(t) : 0.f);
        }
        ++count;
        break;
      }
      if (!DRAFT && rejected > 0) {      // without the rejected tokens
        bool hit = false;
        for (int k = 0; k < rejected; ++k) {
          const int g = (gone[k] + z.shift) / VEC;
          hit |= g >= g0 && g < g1;
        }
        take(hit ? sum_rest(rejected) : share[me]);
      }
      if (rejected == 0 || !(total > 0.0)) {      // (nothing is left: from p itself)
        rejected = 0;
        total = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          mine[k] = share[lane * 4 + k];
          total += mine[k];
        }
        total = warp_sum_d(total);
      }
      const double aim = static_cast<double>(num[0]) * total;
      double run = (mine[0] + mine[1]) + (mine[2] + mine[3]);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += v;
      }
      double before = __shfl_up_sync(0xffffffffu, run, 1), start = 0.0;
      if (lane == 0) before = 0.0;
      int owner = -1, last = -1;      // the first part that passes, the last that has something
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (mine[k] > 0.0) {
          last = lane * 4 + k;
          if (owner < 0 && before + mine[k] > aim) {
            owner = lane * 4 + k;
            start = before;
          }
        }
        before += mine[k];
      }
      const unsigned over = __ballot_sync(0xffffffffu, owner >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
      if (over) {
        const int l = __ffs(over) - 1;
        owner = __shfl_sync(0xffffffffu, owner, l);
        start = __shfl_sync(0xffffffffu, start, l);
      } else {      // a number of 1 and more, or none: the last token that has a share
        owner = __shfl_sync(0xffffffffu, last, 31 - __clz(any));
        start = 0.0;
      }
      if (me == owner) {
        int hit = -1, end = 0;
        each([&](int g, const uint4 (&wz)[LOADS], const uint4 (&wd)[DRAFT ? LOADS : 1]) {
#pragma unroll 1
          for (int u = 0; u < LOADS; ++u) {
            const int e = (g + u * 32 + lane) * VEC - z.shift;
            const uint4 x = wz[u], y = wd[DRAFT ? u : 0];
            double w[VEC], own = 0.0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              w[i] = rest(e + i, Row::element(x, i), DRAFT ? Row::element(y, i) : 0.f, rejected);
              own += w[i];
            }
            double sofar = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double v = __shfl_up_sync(0xffffffffu, sofar, o);
              if (lane >= o) sofar += v;
            }
            double at_lane = __shfl_up_sync(0xffffffffu, sofar, 1);
            if (lane == 0) at_lane = 0.0;
            at_lane += start;
            int pass = -1, has = -1;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              at_lane += w[i];
              if (w[i] > 0.0) {
                has = e + i;
                if (pass < 0 && over && at_lane > aim) pass = e + i;
              }
            }
            const unsigned passed = __ballot_sync(0xffffffffu, pass >= 0), there = __ballot_sync(0xffffffffu, has >= 0);
            if (there) end = __shfl_sync(0xffffffffu, has, 31 - __clz(there));
            if (passed) {
              hit = __shfl_sync(0xffffffffu, pass, __ffs(passed) - 1);
              return false;
            }
            start += __shfl_sync(0xffffffffu, sofar, 31);
          }
          return true;
        });
        if (hit < 0) hit = end;
        if (lane == 0) {
          a.out_tokens[out + count] = hit;
          a.out_logprobs[out + count] = logprob(z.at(hit));
        }
      }
      ++count;
      break;
    }
  }
  if (rank == 0) {
    if (tid == 0) a.out_counts[b] = count;
    for (int i = count + tid; i < a.steps; i += DV_THREADS) {
      a.out_tokens[out + i] = -1;
      a.out_rows[out + i] = -1;
      a.out_logprobs[out + i] = 0.f;
    }
  }
}

template <typename T, bool DRAFT>
int launch_verify(const VerifyArgs& a, int B, cudaStream_t stream) {
  // Two CTAs to an SM. The largest cluster with which all sequences run at once.
  int dev = 0, sms = 148;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  int cluster = DV_CLUSTER;
  while (cluster > 1 && static_cast<long long>(B) * cluster > 2 * sms) cluster /= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B) * cluster);
  cfg.blockDim = dim3(DV_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = cluster;
  attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = rlb_pdl_enabled() ? 2 : 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, verify_kernel<T, DRAFT>, a));
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
  if (static_cast<long long>(B) * DV_CLUSTER > 0x7fffffffll) return -2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (f32) return draft ? launch_verify<float, true>(a, B, st) : launch_verify<float, false>(a, B, st);
  return draft ? launch_verify<__nv_bfloat16, true>(a, B, st) : launch_verify<__nv_bfloat16, false>(a, B, st);
}
