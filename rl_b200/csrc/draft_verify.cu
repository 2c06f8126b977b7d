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
// One CTA per sequence (and one for the rows before the first and behind the last), a thread per row: it walks up its parents. Every row is written by one CTA, whatever the offsets are: a
// sequence's begin at the largest offset up to its own.
__global__ void __launch_bounds__(DR_ROWS)
tree_rows_kernel(const int* __restrict__ parents, const int* __restrict__ cu, const int* __restrict__ ctx, const int* __restrict__ table, long long table_ld,
                 int pages, int block, int B, int T, int max_rows, int words, int* __restrict__ masks, int* __restrict__ positions,
                 long long* __restrict__ slots, int* status) {
  __shared__ int up[DR_ROWS], before[DR_ROWS / 32];
  pdl_sync();
  const int b = blockIdx.x, j = threadIdx.x;
  auto none = [&](int from, int to) {      // rows of no sequence see nothing and have no place
    for (long long t = from + j; t < to; t += blockDim.x) {
      for (int w = 0; w < words; ++w) masks[t * words + w] = 0;
      positions[t] = 0;
      slots[t] = -1;
    }
  };
  int own = 0;
  for (int i = j; i <= b; i += DR_ROWS) own = max(own, cu[i]);
  own = __reduce_max_sync(0xffffffffu, own);
  if ((j & 31) == 0) before[j >> 5] = own;
  const TreeSpan s = b < B ? tree_span(cu, b, T, max_rows, status, j == 0) : TreeSpan{0, 0};
  if (j < s.n) {
    const int p = parents[s.lo + j];
    up[j] = p >= 0 && p < j ? p : -1;
    if ((p >= j || p < -1) && status) atomicCAS(status, 0, RLB_ERR_BOUNDS);
  }
  __syncthreads();
  own = 0;
#pragma unroll
  for (int w = 0; w < DR_ROWS / 32; ++w) own = max(own, before[w]);
  own = min(own, T);
  if (b == B) {
    none(0, min(max(cu[0], 0), T));
    none(own, T);
    return;
  }
  none(max(s.lo + s.n, own), min(max(cu[b + 1], s.lo), T));      // (rows over max_rows)
  if (j >= s.n || s.lo + j < own) return;
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
// distribution over 10^5 tokens would be off by as much as a token has. A weight is 2^(l c - N), c = log2(e) / T, with a whole number N next to the largest l c that a warp has met first: so
// sums of several warps are joined by their exponents. l c - N is cut into 256ths, a table's entry, and a rest r, |r| <= 1 / 512, for which a polynomial of third degree is off by
// (r ln 2)^4 / 24 < 1.5e-13. Eight instructions of the 64-bit pipe a logit and, with the loads,
// some twenty others.
//
// A cluster of CTAs has a sequence. It walks down the accepted rows and reads the logits of these rows alone, which is what the operator cannot do without: each warp has a range
// of tokens and leaves its sum in every CTA's shared memory; all CTAs come to the same decision. The ranges' sums say in which range the last token lies, whose CTA
// goes through it once more. With draft logits the sums are taken again behind a rejection; without, the rejected tokens' weights are taken off their ranges.
//
// Bound by the instructions' rate (64 trees of 17 rows, 128256 logits: 52 us for 56 MB, 58 % of the issue slots while an SM has work) and by latency: a row is its sums (5500 cycles of
// 11000), the exchange (1400), the joining of the parts (1000) and the children (1000), one after another; a single row of 128256 logits takes 10 us, a chain of 6 with 32000 logits 10.
// 48 sequences of 8 drawn rows, 151936 logits: 127 us for 82 MB. A first pass in 32 bits with sums in 64 where they decide was slower, so were 256 threads in clusters of 16, a table
// entry for each of 128ths in 16 copies without conflicts of banks, eight loads of a lane on their way in place of four, and the first child's logits fetched while a row's parts are exchanged.
// What the functions behind a row's sums read lies in shared memory: in every thread's own memory (52 KB a CTA) it came from the second level cache (59 us in place of 52).
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
constexpr int DV_ELEMS = 8;      // logits a lane has at a time
constexpr int DV_SLOTS = 4;      // loads of 16 bytes that a lane has on their way (eight are no faster)
constexpr int EXP_STEPS = 256;
constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.69314718055994530942;
constexpr double MAGIC = 6755399441055744.0 / EXP_STEPS;      // 1.5 * 2^52 / 256: a sum with it has the nearest number of 256ths in its low word
constexpr float F_MAX = 3.402823466e38f;
// Two probabilities are off by up to 3e-13 from one another, relatively, where they are equal: a draft's are taken as 4.5e-13 more, so that nothing is left of tokens that are as probable in both.
constexpr double DRAFT_MORE = 1.0 + 0x1p-41;
constexpr float COLDEST = 1.17549435e-38f;      // temperatures below are greedy

// Copies of 16 bytes to shared memory, which the lane that issued them reads itself.
__device__ __forceinline__ void copy16(uint4* to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// NaN weighs nothing, +inf as much as the largest number.
__device__ __forceinline__ float usable(float x) { return fminf(fmaxf(x, -INFINITY), F_MAX); }
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float max3(float a, float b, float c) {      // of those that are numbers
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float warp_top(float x) {      // largest of the warp's numbers, none of them NaN
  const int u = __float_as_int(x), m = __reduce_max_sync(0xffffffffu, u < 0 ? u ^ 0x7fffffff : u);
  return __int_as_float(m < 0 ? m ^ 0x7fffffff : m);
}
// x in 64 bits times 2^-896, by its bits (the conversion instruction gives one lane a cycle).
__device__ __forceinline__ double lowered(float x) {
  const int u = __float_as_int(x);
  return __hiloint2double((u >> 3) & 0x8fffffff, u << 29);
}
// 2^z of |z| <= 1022 as table entry, rest and exponent: `t` is z + MAGIC, `r` what z has over its 256ths.
__device__ __forceinline__ double power(const double* table, double t, double r) {
  const int k = __double2loint(t);
  const double p = r * (LN2 + r * (LN2 * LN2 / 2 + r * (LN2 * LN2 * LN2 / 6)));
  const double f = table[k & (EXP_STEPS - 1)];      // without what its index adds to the exponent below
  const double s = __hiloint2double(__double2hiint(f) + k * (0x100000 / EXP_STEPS), __double2loint(f));
  return fma(s, p, s);
}
// log2 of a sum: 32 bits, then one step on 2^-l s = 1 + d.
__device__ __noinline__ double log2_of(const double* table, double s) {
  const int hi = __double2hiint(s), e = (hi >> 20) - 1023;
  const double f = __hiloint2double((hi & 0xfffff) | 0x3ff00000, __double2loint(s));
  const double l = static_cast<double>(__log2f(static_cast<float>(f))), t = MAGIC - l, d = fma(f, power(table, t, -l - (t - MAGIC)), -1.0);
  return e + (l + (d - d * d * 0.5 + d * d * d * (1.0 / 3)) * LOG2E);
}

struct Temperature {
  double c;            // log2(e) / T * 2^896
  float far, near;     // differences of logits that make 2^1000 and 2^60, rounded down
};
// Weights relative to 2^N, N = rint(top c). A logit that is less than 2^-1000 of the row's largest weighs nothing.
struct Frame {
  double add;          // MAGIC - N
  float top, low;      // logits below `low` weigh nothing (2^-1000 of top's)
  int kind;            // 0: what is below `low` may be taken as `low` in a sum; 1: it may not; 2: so far apart are the logits (top c beyond 2^42) that top's equals alone have weight
  static __device__ __noinline__ Frame frame_of(float x, const Temperature q) {
    Frame f;
    f.set(x, q);
    return f;
  }
  __device__ __forceinline__ void set(float x, const Temperature q) {
    top = x;
    low = fmaxf(fminf(__fsub_ru(x, q.far), x), -F_MAX);
    const double m = lowered(x) * q.c, n = (m + 256 * MAGIC) - 256 * MAGIC;
    add = MAGIC - n;
    kind = !(fabs(m) < 0x1p42) ? 2 : low >= x || low <= -F_MAX ? 1 : 0;
  }
  // `v` in a frame with a larger N
  static __device__ __forceinline__ double moved(double v, double add, double larger) {
    const double d = larger - add, scaled = v * __hiloint2double((1123 + __double2loint(d + 256 * MAGIC)) << 20, 0) * 0x1p-100;
    return static_cast<uint32_t>(__double2hiint(d)) <= 0xc090e000u ? scaled : 0.0;      // (-1080)
  }
  __device__ __forceinline__ void move(float x, const Temperature& q, double& total) {
    const Frame before = *this;
    *this = frame_of(x, q);
    total = before.top == -INFINITY ? 0.0 : moved(total, before.add, add);
  }
  __device__ __forceinline__ double depth(double c, float x) const { return kind == 2 ? 0.0 : fma(lowered(x), c, add - MAGIC); }      // x c - N
  __device__ __forceinline__ double near(const double* table, double c, float x) const {
    const double v = lowered(x), t = fma(v, c, add);
    return power(table, t, fma(v, c, add - t));
  }
};

// One weight in a frame of any kind.
__device__ __forceinline__ double weight_of(const Frame& f, const double* table, double c, float x) {
  const double near = f.near(table, c, fminf(fmaxf(x, f.low), f.top));
  return !(x >= f.low) ? 0.0 : f.kind == 2 ? (x == f.top ? 1.0 : 0.0) : near;
}
__device__ __forceinline__ void push_u(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void push_row(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void push_d(uint32_t addr, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory"); }

struct __align__(16) TreeRow {
  int up, token;
  float number, z;      // z: of a child of the visited row, its token's logit there
};
// Of the warps' ranges, target or draft: sum of weights in its frame, the frame's MAGIC - N, the range's largest logit (-inf: none) and, where that is asked for, its place.
// A lane that joins has four ranges beside one another: these lie in as many rows.
struct Parts {
  double sum[DV_PARTS], add[DV_PARTS];
  float peak[DV_PARTS];
  int at[DV_PARTS];
};
__device__ __forceinline__ int part_place(int w) { return (w & 3) * 32 + (w >> 2); }

template <typename T>
struct RowLogits {
  static constexpr int VEC = 16 / sizeof(T), LOADS = DV_ELEMS / VEC;
  const T* p;
  int V;
  int shift;      // elements before the row's first that its first group of 16 bytes has
  bool vec;
  bool inner;     // all of this warp's range lies on 16 bytes and within the row
  __device__ __forceinline__ void range(int g0, int g1) { inner = vec && g0 * VEC >= shift && g1 * VEC - shift <= V; }
  // Group g's elements, g * VEC - shift and on, to the lane's place in shared memory; those behind group g1 or outside of the row are -inf.
  __device__ __forceinline__ void stage(uint4* to, int g, int g1) const {
    const int e = g * VEC - shift;
    if (g >= g1) {
      constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
      *to = make_uint4(none, none, none, none);
    } else if (inner || (vec && e >= 0 && e + VEC <= V)) {
      copy16(to, p + e);
    } else {
      *to = edge(p, e, V);
    }
  }
  static __device__ __noinline__ uint4 edge(const T* p, int e, int V) {      // (a call waits for what it loads)
    uint4 v;
    uint32_t* w = &v.x;
    if (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = e + i >= 0 && e + i < V ? reinterpret_cast<const uint32_t*>(p)[e + i] : 0xff800000u;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int a = e + 2 * i;
        const uint32_t lo = a >= 0 && a < V ? reinterpret_cast<const uint16_t*>(p)[a] : 0xff80u;
        const uint32_t hi = a + 1 >= 0 && a + 1 < V ? reinterpret_cast<const uint16_t*>(p)[a + 1] : 0xff80u;
        w[i] = lo | hi << 16;
      }
    }
    return v;
  }
  static __device__ __forceinline__ float raw(const uint4& v, int i) { return raw(&v.x, i); }
  static __device__ __forceinline__ float raw(const uint32_t* w, int i) {
    return sizeof(T) == 4 ? __uint_as_float(w[i]) : __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
  static __device__ __forceinline__ float element(const uint4& v, int i) { return usable(raw(v, i)); }
  static __device__ __noinline__ double seldom(uint4 v, Frame f, const double* table, double c) {      // a group's weights in frames of the other kinds
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float x = element(v, i);
      t += !(x >= f.low) ? 0.0 : f.kind == 2 ? (x == f.top ? 1.0 : 0.0) : f.near(table, c, x);
    }
    return t;
  }
  __device__ __forceinline__ float at(int i) const { return usable(static_cast<float>(p[i])); }
};

struct RowSum {      // of all parts
  Frame f;
  double inv, sum;      // the sum's reciprocal (0: no logit above -inf)
};

// A visited row: its logits, the draft's, and what its sums and rejections came to (in shared memory).
template <typename T, bool DRAFT>
struct Visit {
  RowLogits<T> z, d;
  const RowSum* row;      // [1 + DRAFT]
  const double* table;
  const double* grow;
  const int* gone;
  uint4* slots;      // of all lanes, DV_THREADS apart
  double c;
};
// What is left of the probability of token i after `r` rejections, from its logits.
template <typename T, bool DRAFT>
__device__ __noinline__ double rest_of(const Visit<T, DRAFT>& v, int i, float x, float y, int r) {
  double w = weight_of(v.row[0].f, v.table, v.c, x) * v.row[0].inv;
  if (r == 0) return w;
  if (DRAFT) {
    const Frame& f = v.row[DRAFT].f;      // (what is below `low` as much as that, where sum_left may be asked for the same)
    const double g = (f.kind == 0 ? f.near(v.table, v.c, fminf(fmaxf(y, f.low), f.top)) : weight_of(f, v.table, v.c, y)) * v.row[DRAFT].inv;
#pragma unroll 1
    for (int k = 0; k < r; ++k) w = fmax(fma(w, v.grow[k], -g), 0.0);
  } else {
#pragma unroll 1
    for (int k = 0; k < r; ++k) w = v.gone[k] == i ? 0.0 : w;
  }
  return w;
}
// The same of the tokens from e0 to e1, summed over the warp.
template <typename T, bool DRAFT>
__device__ __noinline__ double sum_of(const Visit<T, DRAFT>& v, int e0, int e1, int r) {
  double sum = 0.0;
  int e = e0 + (threadIdx.x & 31);
  float x[4], y[4];
  auto fetch = [&](int from) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = from + 32 * k;
      x[k] = i < e1 ? v.z.at(i) : -INFINITY;
      y[k] = DRAFT && i < e1 ? v.d.at(i) : 0.f;
    }
  };
  const Frame f = v.row[0].f;
  if (f.kind == 0 && (!DRAFT || r == 0)) {      // as in the row's own sums
    const double inv = v.row[0].inv, c = v.c;
    const double* table = v.table;
#pragma unroll 1
    for (; e < e1; e += 128) {
      fetch(e);
      double w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = x[k] >= f.low ? f.near(table, c, x[k]) : 0.0;
#pragma unroll 1
      for (int g = 0; g < r; ++g) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = v.gone[g] == e + 32 * k ? 0.0 : w[k];
      }
      sum += (w[0] + w[1]) + (w[2] + w[3]);
    }
    __syncwarp();
    return warp_sum_d(sum) * inv;
  }
#pragma unroll 1
  for (; e < e1; e += 128) {
    fetch(e);
    sum += rest_of<T, DRAFT>(v, e, x[0], y[0], r);
    if (e + 32 < e1) sum += rest_of<T, DRAFT>(v, e + 32, x[1], y[1], r);
    if (e + 64 < e1) sum += rest_of<T, DRAFT>(v, e + 64, x[2], y[2], r);
    if (e + 96 < e1) sum += rest_of<T, DRAFT>(v, e + 96, x[3], y[3], r);
  }
  __syncwarp();
  return warp_sum_d(sum);
}
// The same of the groups from g0 to g1 of a row and its draft's, both of kind 0 and without infinities: as in the row's own sums, but that what weighs nothing in the target is nothing, or a
// difference would be left where no token has a share and the last token could fall there. (2^-500 and less, `low`'s weight, times a factor without exponent, below 2^-1042, is zero: 127 us for 48 of
// 8 drawn rows, 151936 logits, as without it; 131 with the weight itself chosen.) The draft's is at least `low`'s, here and in rest_of.
template <typename T>
__device__ __noinline__ double sum_left(const Visit<T, true>& v, int g0, int g1, int r) {
  constexpr int VEC = RowLogits<T>::VEC;
  const int lane = threadIdx.x & 31;
  RowLogits<T> z = v.z, d = v.d;
  z.range(g0, g1);
  d.range(g0, g1);
  const Frame p = v.row[0].f, q = v.row[1].f;
  const double inv = v.row[0].inv, dinv = v.row[1].inv, c = v.c;
  const double* table = v.table;
  double even = 0.0, odd = 0.0;
  constexpr int AHEAD = DV_SLOTS / 2;
  uint4* to = v.slots + threadIdx.x;
#pragma unroll 1
  for (int k = 0; k < AHEAD; ++k, to += 2 * DV_THREADS) {
    z.stage(to, g0 + 32 * k + lane, g1);
    d.stage(to + DV_THREADS, g0 + 32 * k + lane, g1);
    copies_commit();
  }
  int at = 0;
#pragma unroll 1
  for (int g = g0; g < g1; g += 32) {
    copies_wait<AHEAD - 1>();
    to = v.slots + threadIdx.x + at * (2 * DV_THREADS);
    const uint32_t *xs = reinterpret_cast<const uint32_t*>(to), *ys = reinterpret_cast<const uint32_t*>(to + DV_THREADS);
#pragma unroll 1
    for (int h = 0; h < VEC; h += 4, xs += sizeof(T), ys += sizeof(T)) {      // four at a time: more do not fit the registers
      double w[4], e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = RowLogits<T>::raw(xs, i);
        w[i] = p.near(table, c, fmaxf(x, p.low)) * __hiloint2double(x >= p.low ? __double2hiint(inv) : 0, __double2loint(inv));
        e[i] = q.near(table, c, fmaxf(RowLogits<T>::raw(ys, i), q.low)) * dinv;
      }
#pragma unroll 1
      for (int k = 0; k < r; ++k) {
        const double grow = v.grow[k];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = fmax(fma(w[i], grow, -e[i]), 0.0);
      }
      even += w[0] + w[2];
      odd += w[1] + w[3];
    }
    at = (at + 1) % AHEAD;
    if (g + 32 * AHEAD < g1) {
      z.stage(to, g + 32 * AHEAD + lane, g1);
      d.stage(to + DV_THREADS, g + 32 * AHEAD + lane, g1);
    }
    copies_commit();
  }
  __syncwarp();
  return warp_sum_d(even + odd);
}
// The token of [e0, e1) at which the running sum from `start` passes `aim` (none: the last with a share; -1: none has). By a warp.
template <typename T, bool DRAFT>
__device__ __noinline__ int find_token(const Visit<T, DRAFT>& v, int e0, int e1, int r, double start, double aim, bool inside) {
  const int lane = threadIdx.x & 31;
  int last = -1;
#pragma unroll 1
  for (int e = e0; e < e1; e += 32) {
    const int i = e + lane;
    const double w = i < e1 ? rest_of<T, DRAFT>(v, i, v.z.at(i), DRAFT ? v.d.at(i) : 0.f, r) : 0.0;
    __syncwarp();
    double run = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u;
    }
    const unsigned over = __ballot_sync(0xffffffffu, inside && w > 0.0 && start + run > aim), any = __ballot_sync(0xffffffffu, w > 0.0);
    if (over) return e + __ffs(over) - 1;
    if (any) last = e + 31 - __clz(any);
    start += __shfl_sync(0xffffffffu, run, 31);
  }
  return last;
}

template <typename T, bool DRAFT>
__global__ void __launch_bounds__(DV_THREADS, 2)
verify_kernel(const VerifyArgs a) {
  using Row = RowLogits<T>;
  constexpr int VEC = Row::VEC, LOADS = Row::LOADS, STEP = 32 * LOADS, AHEAD = 2;
  extern __shared__ uint4 ring[];                     // [AHEAD steps][LOADS][DV_THREADS]
  __shared__ double table[EXP_STEPS];
  __shared__ Parts parts[2][1 + DRAFT];      // of all warps of the cluster, by turns
  __shared__ double share[DV_PARTS], pieces[DV_WARPS];      // the ranges' probabilities; sums of a range's pieces
  __shared__ RowSum row[1 + DRAFT];
  __shared__ int row_best;
  __shared__ TreeRow tree[DR_ROWS];
  __shared__ float ld[DR_ROWS];      // as TreeRow::z, the draft's
  __shared__ int gone[DR_ROWS];
  __shared__ double left[DR_ROWS + 1], grow[DR_ROWS + 1];       // what is left to be given after so many rejections; its reciprocal, without draft logits the rejected tokens' weights
  __shared__ double chosen[DR_ROWS], sums[DR_ROWS];             // of each accepted step: l c - N of its token, the sum of weights
  __shared__ int verdict, tried, turned_down;
  __shared__ Visit<T, DRAFT> visit;
  // (A shuffle or a vote where the compiler cannot rule out that the warp's lanes have parted costs some 260 cycles in place of 20: what decides on loops and branches goes
  // through one first.)
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  uint32_t ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int rank = static_cast<int>(cluster_ctarank()), b = blockIdx.x / ctas, W = static_cast<int>(ctas) * DV_WARPS, me = rank * DV_WARPS + warp;
  if (tid < EXP_STEPS) {      // 2^(i / 256) by exp's series, 0.7^18 / 18! < 3e-19
    const double y = tid * (LN2 / EXP_STEPS);
    double v = 1.0;
#pragma unroll
    for (int i = 17; i > 0; --i) v = fma(v, y * (1.0 / i), 1.0);
    table[tid] = __hiloint2double(__double2hiint(v) - tid * (0x100000 / EXP_STEPS), __double2loint(v));
  }
  __syncthreads();
  pdl_sync();
  const TreeSpan span = tree_span(a.cu, b, a.T, a.max_rows, a.status, tid == 0 && rank == 0), s{__shfl_sync(0xffffffffu, span.lo, 0), __shfl_sync(0xffffffffu, span.n, 0)};
  const long long out = static_cast<long long>(b) * a.steps;
  int count = 0, drawn = -1;      // the last token, of the thread that has it
  float drawn_z = 0.f;
  double depth_c = 0.0;
  if (s.n > 0) {
    const float given = a.temps ? a.temps[b] : static_cast<float>(a.temp);
    const bool cold = __any_sync(0xffffffffu, a.greedy || !(given >= COLDEST));
    const double temp = !(given >= COLDEST) ? 1.0 : a.temps ? static_cast<double>(given) : a.temp;
    const Temperature tp{LOG2E / temp * 0x1p896, __double2float_rd(1000 * LN2 * temp), __double2float_rd(60 * LN2 * temp)};
    const int groups_per = (a.V + 2 * VEC - 2) / VEC / W + 1;      // groups of a range, whatever the row's alignment
    depth_c = tp.c;
    int turn = 0, node = 0, own_up = -1, own_tok = -1;
    float own_num = 0.f;
    bool started = false;
    cluster_arrive();

    auto begin = [&]() {
      turn ^= 1;
      if (!started) cluster_wait();      // (all CTAs of the cluster run before one writes into another's memory)
      started = true;
    };
    auto push = [&](int which, double sum, double add, float peak, int at) {      // this warp's part to all CTAs
      if (lane < static_cast<int>(ctas)) {
        Parts& to = parts[turn][which];
        const int place = part_place(me);
        push_d(mapa_shared(smem_u32(&to.sum[place]), lane), sum);
        push_d(mapa_shared(smem_u32(&to.add[place]), lane), add);
        push_u(mapa_shared(smem_u32(&to.peak[place]), lane), __float_as_uint(peak));
        if (cold) push_u(mapa_shared(smem_u32(&to.at[place]), lane), static_cast<uint32_t>(at));
      }
    };
    auto end = [&]() {
      cluster_arrive();
      cluster_wait();
    };

    while (true) {
      const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(static_cast<const T*>(a.logits) + (s.lo + node) * a.ld) % 16 / sizeof(T));
      const int groups = (a.V + shift + VEC - 1) / VEC, g0 = min(groups, me * groups_per), g1 = min(groups, g0 + groups_per);
      auto row_of = [&](int which) {      // the target's, the draft's (made again where it is asked for: registers are short)
        Row r{static_cast<const T*>(DRAFT && which ? a.draft : a.logits) + (s.lo + node) * (DRAFT && which ? a.ld_draft : a.ld), a.V, shift, false, false};
        r.vec = reinterpret_cast<uintptr_t>(r.p) % 16 / sizeof(T) == shift;
        r.range(g0, g1);
        return r;
      };
      auto stage = [&](const Row& r, uint4* to, int g) {      // of a step
#pragma unroll
        for (int u = 0; u < LOADS; ++u) r.stage(to + u * DV_THREADS, g + u * 32 + lane, g1);
      };
      auto first_steps = [&](const Row& r) {
#pragma unroll 1
        for (int k = 0; k < AHEAD; ++k) {
          if (g0 + k * STEP < g1) stage(r, ring + tid + k * (LOADS * DV_THREADS), g0 + k * STEP);
          copies_commit();
        }
      };
      // The tree and its children's logits are read by the first CTA alone, for all: what the CTAs decide comes from the same numbers even where another stream is writing them.
      const bool mine_of_tree = rank == 0 && tid < s.n, first_row = count == 0;
      if (first_row && mine_of_tree) {
        own_up = tid ? a.parents[s.lo + tid] : -1;
        own_tok = a.tokens[s.lo + tid];
        own_num = a.uniforms[s.lo + tid];
      }
      first_steps(row_of(0));
      if (tid == 0) visit = Visit<T, DRAFT>{row_of(0), DRAFT ? row_of(1) : Row{}, row, table, grow, gone, ring, tp.c};      // (read behind this row's barrier)
      const bool child = mine_of_tree && tid > node && own_up == node && own_tok >= 0 && own_tok < a.V;
      T own_z{}, own_d{};      // (waited for where they are passed on)
      if (child) {
        own_z = row_of(0).p[own_tok];
        if (DRAFT) own_d = row_of(1).p[own_tok];
      }
      // ---------------------------------------------------------------- the sums of the row, the target's and then the draft's
      begin();
#pragma unroll 1
      for (int which = 0; which < (DRAFT && !cold ? 2 : 1); ++which) {
        const Row r = row_of(which);
        float peak = -INFINITY;      // the largest that a lane has met first
        int at = 0x7fffffff;
        Frame f;
        f.top = -INFINITY;
        float high = -INFINITY, most = -INFINITY;
        double sum = 0.0;
        int slot = 0;
#pragma unroll 1
        for (int g = g0; g < g1; g += STEP) {
          copies_wait<AHEAD - 1>();
          uint4* from = ring + tid + slot * (LOADS * DV_THREADS);
          uint4 v[LOADS];
#pragma unroll
          for (int u = 0; u < LOADS; ++u) v[u] = from[u * DV_THREADS];
          slot = (slot + 1) % AHEAD;
          if (g + AHEAD * STEP < g1) stage(r, from, g + AHEAD * STEP);
          copies_commit();
          if (cold) {
#pragma unroll
            for (int u = 0; u < LOADS; ++u)
#pragma unroll
              for (int i = 0; i < VEC; ++i) {
                const float x = Row::element(v[u], i);
                if (x > peak) {
                  peak = x;
                  at = (g + u * 32 + lane) * VEC - r.shift + i;
                }
              }
          }
          float top = -INFINITY;
#pragma unroll
          for (int u = 0; u < LOADS; ++u)
#pragma unroll
            for (int i = 0; i < VEC; i += 2) top = max3(top, Row::raw(v[u], i), Row::raw(v[u], i + 1));
          most = fmaxf(most, top);
          if (__any_sync(0xffffffffu, top > high)) {      // the first numbers, or some that weigh 2^60 and more
            top = fminf(warp_top(top), F_MAX);
            if (top > f.top) {
              f.move(top, tp, sum);
              high = fmaxf(__fadd_rd(top, tp.near), top);
            }
          }
          if (f.top == -INFINITY) continue;
          if (f.kind != 0 || high >= F_MAX) {      // (F_MAX: there may be +inf)
#pragma unroll
            for (int u = 0; u < LOADS; ++u) sum += Row::seldom(v[u], f, table, tp.c);
            continue;
          }
          double even = 0.0, odd = 0.0;      // what is below `low`, and what is not a number, is taken as 2^-1000
#pragma unroll
          for (int u = 0; u < LOADS; ++u)
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
              even += f.near(table, tp.c, fmaxf(Row::raw(v[u], i), f.low));
              odd += f.near(table, tp.c, fmaxf(Row::raw(v[u], i + 1), f.low));
            }
          sum += even + odd;
        }
        if (DRAFT && which == 0 && !cold) first_steps(row_of(1));
        __syncwarp();
        sum = warp_sum_d(sum);
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
        push(which, sum, f.add, fminf(warp_top(most), F_MAX), at);
      }
      if (mine_of_tree && (first_row || child))
        for (uint32_t to = 0; to < ctas; ++to) {
          const uint32_t at = mapa_shared(smem_u32(&tree[tid]), to);
          if (first_row) push_row(at, static_cast<uint32_t>(own_up), static_cast<uint32_t>(own_tok), __float_as_uint(own_num), __float_as_uint(usable(static_cast<float>(own_z))));
          if (child) {
            if (!first_row) push_u(at + 12, __float_as_uint(usable(static_cast<float>(own_z))));
            if (DRAFT) push_u(mapa_shared(smem_u32(&ld[tid]), to), __float_as_uint(usable(static_cast<float>(own_d))));
          }
        }
      end();
      // a warp joins the target's parts, another the draft's: lane i has four of them, in their order
      if (warp < 1 + DRAFT) {
        const Parts& got = parts[turn][warp];
        RowSum& to = row[warp];
        float m[4], top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          m[k] = lane * 4 + k < W ? got.peak[k * 32 + lane] : -INFINITY;
          top = fmaxf(top, m[k]);
        }
        const Frame whole = Frame::frame_of(warp_top(top), tp);
        double v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {      // of rows with one logit far above the others the parts that have it
          const double sum = got.sum[k * 32 + lane], moved = Frame::moved(sum, got.add[k * 32 + lane], whole.add);
          v[k] = !(m[k] >= whole.low) ? 0.0 : whole.kind == 2 ? (m[k] == whole.top ? sum : 0.0) : moved;
        }
        const double all = warp_sum_d((v[0] + v[1]) + (v[2] + v[3])), inv = whole.top > -INFINITY && !(cold && warp) ? 1.0 / all : 0.0;
        if (warp == 0)
#pragma unroll
          for (int k = 0; k < 4; ++k) share[k * 32 + lane] = v[k] * inv;
        int best = -1;
        if (cold && warp == 0 && whole.top > -INFINITY) {      // the first range that has the largest (ranges lie in the tokens' order)
#pragma unroll
          for (int k = 3; k >= 0; --k) best = m[k] == whole.top ? got.at[k * 32 + lane] : best;
        }
        if (cold) best = __shfl_sync(0xffffffffu, best, max(0, __ffs(__ballot_sync(0xffffffffu, best >= 0)) - 1));
        if (lane == 0) {
          to.f = whole;
          to.inv = DRAFT && warp ? inv * DRAFT_MORE : inv;
          to.sum = all;
          if (warp == 0) {
            if (cold) row_best = max(0, best);
            left[0] = grow[0] = 1.0;
            tried = node;
            turned_down = 0;
          }
        }
        __syncwarp();
      }
      if (DRAFT) __syncthreads();
      const int e0 = max(0, g0 * VEC - shift), e1 = min(a.V, g1 * VEC - shift);      // the range's tokens
      double mine[4], total = 0.0;
      auto take = [&](double v) {      // this warp's part of new sums; the parts and the whole sum of all
        begin();
        push(0, v, 0.0, 0.f, 0);
        end();
#pragma unroll
        for (int k = 0; k < 4; ++k) mine[k] = lane * 4 + k < W ? parts[turn][0].sum[k * 32 + lane] : 0.0;
        total = warp_sum_d((mine[0] + mine[1]) + (mine[2] + mine[3]));
      };
      // ---------------------------------------------------------------- the children
      int next = -1, rejected = 0;
      while (true) {
        if (warp == 0) {      // verdict: an accepted row, -1 none, -2 one rejected after which the sums are taken again
          int v = -1, r = rejected, j0 = tried + 1, stop = s.n;      // 32 rows at a time, each lane has the weight of its own
          double rest = left[r];
          for (int c0 = j0 & ~31; __any_sync(0xffffffffu, c0 < s.n && v == -1 && count + 1 < a.steps); c0 += 32) {
            const int j = c0 + lane, t = j < s.n ? tree[j].token : -1;
            const bool child = j >= j0 && j < s.n && tree[j].up == node && t >= 0 && t < a.V;      // (others have no probability, and are none of the draft's)
            unsigned todo = __ballot_sync(0xffffffffu, child);
            if (todo == 0) continue;
            if (cold) {
              todo = __ballot_sync(0xffffffffu, child && row[0].inv > 0.0 && t == row_best);
              if (todo) v = c0 + __ffs(todo) - 1;
              continue;
            }
            const float x = child ? tree[j].z : -INFINITY, y = DRAFT && child ? ld[j] : -INFINITY;
            double w = rest_of<T, DRAFT>(visit, t, x, y, r), asked = child ? static_cast<double>(tree[j].number) : 0.0;
            if (DRAFT) asked *= weight_of(row[DRAFT].f, table, tp.c, y) * row[DRAFT].inv;
            __syncwarp();
            for (; todo; todo &= todo - 1) {
              const int l = __ffs(todo) - 1, tl = __shfl_sync(0xffffffffu, t, l);
              const double wl = __shfl_sync(0xffffffffu, w, l), al = __shfl_sync(0xffffffffu, asked, l);
              if (__any_sync(0xffffffffu, al * rest < wl)) {
                v = c0 + l;
                break;
              }
              if (DRAFT) {
                v = -2;
                stop = c0 + l;
                break;
              }
              if (__any_sync(0xffffffffu, wl > 0.0)) {
                rest -= wl;
                if (lane == 0) {
                  gone[r] = tl;
                  grow[r] = wl;
                  left[r + 1] = rest;
                }
                ++r;
                if (t == tl) w = 0.0;      // (a token that is out)
              }
            }
            __syncwarp();
          }
          if (lane == 0) {
            tried = stop;
            verdict = v;
            if (!DRAFT) turned_down = r;
          }
        }
        __syncthreads();
        const int v = __reduce_max_sync(0xffffffffu, verdict);
        if (!DRAFT) rejected = __reduce_max_sync(0xffffffffu, turned_down);
        if (v != -2) {
          next = v;
          break;
        }
        ++rejected;
        if constexpr (DRAFT) {
          const bool simple = row[0].f.kind == 0 && row[1].f.kind == 0 && row[0].f.top < 0.5f * F_MAX && row[1].f.top < 0.5f * F_MAX;
          take(simple ? sum_left<T>(visit, g0, g1, rejected) : sum_of<T, DRAFT>(visit, e0, e1, rejected));
        }
        if (tid == 0) {
          left[rejected] = total;
          grow[rejected] = 1.0 / total;
        }
        __syncthreads();
        if (__any_sync(0xffffffffu, !(total > 0.0))) break;
      }
      // ---------------------------------------------------------------- the token
      const bool some = __any_sync(0xffffffffu, row[0].inv > 0.0);      // a row without a number above -inf has no probabilities
      if (rank == 0 && tid == 0) a.out_rows[out + count] = node;
      if (next >= 0) {
        if (rank == 0 && tid == 0) {
          a.out_tokens[out + count] = tree[next].token;
          chosen[count] = row[0].f.depth(tp.c, tree[next].z);
          sums[count] = row[0].sum;
        }
        ++count;
        node = next;
        __syncthreads();      // (this row's numbers have been read)
        continue;
      }
      if (cold || !some) {
        if (rank == 0 && tid == 0) {
          drawn = some ? row_best : 0;
          drawn_z = some ? visit.z.at(drawn) : 0.f;
        }
        ++count;
        break;
      }
      if (!DRAFT && rejected > 0) {      // without the rejected tokens
        // Their weights are taken off their ranges' sums, of which no more than ten bits are lost. A range without any other token keeps some 500 roundings of its sum (2^-44 of it), which
        // are no token's weight: where a range has lost all but 2^-40, or is so light that its roundings are coarser, the sums are taken again. So a range that has something has a token.
        bool again = left[rejected] < 1.0 / 1024;
#pragma unroll
        for (int k = 0; k < 4; ++k) mine[k] = share[k * 32 + lane];
        for (int r = 0; r < rejected; ++r) {
          const int w = (gone[r] + shift) / VEC / groups_per;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (w == lane * 4 + k) mine[k] -= grow[r];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) again |= share[k * 32 + lane] > 0.0 && mine[k] < fma(0x1p-40, share[k * 32 + lane], 0x1p-960);
        if (!__any_sync(0xffffffffu, again)) {
          total = warp_sum_d((mine[0] + mine[1]) + (mine[2] + mine[3]));
        } else {
          bool hit = false;
          for (int k = 0; k < rejected; ++k) {
            const int g = (gone[k] + shift) / VEC;
            hit |= g >= g0 && g < g1;
          }
          take(__any_sync(0xffffffffu, hit) ? sum_of<T, DRAFT>(visit, e0, e1, rejected) : share[part_place(me)]);
        }
      }
      if (__any_sync(0xffffffffu, rejected == 0 || !(total > 0.0))) {      // (nothing is left: from p itself)
        rejected = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) mine[k] = share[k * 32 + lane];
        total = warp_sum_d((mine[0] + mine[1]) + (mine[2] + mine[3]));
      }
      __syncwarp();
      const double aim = static_cast<double>(tree[0].number) * total;
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
      }
      if (rank == owner / DV_WARPS) {      // the range once more, by all warps of its CTA
        const int r0 = max(0, min(groups, owner * groups_per) * VEC - shift), r1 = min(a.V, (owner + 1) * groups_per * VEC - shift);
        const int piece = (r1 - r0 + DV_WARPS - 1) / DV_WARPS, q0 = min(r1, r0 + warp * piece), q1 = min(r1, q0 + piece);
        const double own = sum_of<T, DRAFT>(visit, q0, q1, rejected);
        if (lane == 0) pieces[warp] = own;
        __syncthreads();
        __syncwarp();
        const double piece_sum = lane < DV_WARPS ? pieces[lane] : 0.0;
        double upto = piece_sum;
#pragma unroll
        for (int o = 1; o < DV_WARPS; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const int filled = 31 - __clz(__ballot_sync(0xffffffffu, piece_sum > 0.0));      // -1: none
        const int mover = over ? __ffs(__ballot_sync(0xffffffffu, piece_sum > 0.0 && start + upto > aim)) - 1 : -1;
        if (mover >= 0) start += __shfl_sync(0xffffffffu, upto - piece_sum, mover);
        const bool inside = mover >= 0;      // (otherwise the last that has a share)
        if (warp == (inside ? mover : max(filled, 0))) {      // (a token is written, whatever the logits became meanwhile)
          const int hit = max(0, find_token<T, DRAFT>(visit, q0, q1, rejected, start, aim, inside));
          if (lane == 0) {
            drawn = hit;
            drawn_z = visit.z.at(hit);
          }
        }
      }
      ++count;
      break;
    }
  }
  if (drawn >= 0) {
    a.out_tokens[out + count - 1] = drawn;
    a.out_logprobs[out + count - 1] = row[0].inv > 0.0 ? static_cast<float>((row[0].f.depth(depth_c, drawn_z) - log2_of(table, row[0].sum)) * LN2) : -INFINITY;
  }
  if (rank == 0) {
    if (tid == 0) a.out_counts[b] = count;
    __syncthreads();
    for (int i = tid; i < count - 1; i += DV_THREADS) a.out_logprobs[out + i] = static_cast<float>((chosen[i] - log2_of(table, sums[i])) * LN2);
    for (int i = count + tid; i < a.steps; i += DV_THREADS) {
      a.out_tokens[out + i] = -1;
      a.out_rows[out + i] = -1;
      a.out_logprobs[out + i] = 0.f;
    }
  }
}

template <typename T, bool DRAFT>
int launch_verify(const VerifyArgs& a, int B, cudaStream_t stream) {
  // Two CTAs to an SM. The largest cluster with which all sequences run at once, or in two turns where they may go down several rows: the last sequences' rows
  // are what the others wait for (us with two turns and with one: 64 trees of 17 rows 54 and 57, 48 of 8 drawn ones 127 and 142, 256 trees of 5 113 and 145; 64 single rows 26 and 21).
  int dev = 0, sms = 148;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  int cluster = DV_CLUSTER;
  while (cluster > 1 && static_cast<long long>(B) * cluster > (a.steps > 1 ? 4 : 2) * sms) cluster /= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B) * cluster);
  cfg.blockDim = dim3(DV_THREADS);
  cfg.dynamicSmemBytes = DV_SLOTS * DV_THREADS * 16;
  e = cudaFuncSetAttribute(verify_kernel<T, DRAFT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(cfg.dynamicSmemBytes));
  if (e != cudaSuccess) return static_cast<int>(e);
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
  if (max_rows < 1 || max_rows > DR_ROWS || steps < 1 || steps > max_rows || V < 1 || V > 1 << 30) return -2;
  const VerifyArgs a{logits, draft, ld, ld_draft, V, T, max_rows, steps, greedy, tokens, parents, cu, uniforms, temps, temp, out_tokens, out_counts, out_rows,
                     out_logprobs, status};
  if (static_cast<long long>(B) * DV_CLUSTER > 0x7fffffffll) return -2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (f32) return draft ? launch_verify<float, true>(a, B, st) : launch_verify<float, false>(a, B, st);
  return draft ? launch_verify<__nv_bfloat16, true>(a, B, st) : launch_verify<__nv_bfloat16, false>(a, B, st);
}
