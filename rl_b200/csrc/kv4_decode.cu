// Decode attention over the 4-bit key/value cache (kv4.cuh): one query token per sequence, softmax(scale q k^T) v over its cached tokens or the last
// `window` of them. A CTA of four warps takes a sequence and one key/value head with up to eight of its query heads. Few sequences: a cluster of up to eight CTAs
// shares the tokens of each and adds the parts through distributed shared memory. Long ones: as many CTAs as the device holds share all tokens evenly, so that each gets
// a run of whole sequences and a part of one or two, and a second kernel joins the parts (kv4_plan in ops/kv4_ops.py has the choice, both sides measured).
//
// Both products run as 16 x 8 x 16 tensor-core instructions whose 16-row operand comes from the codes in registers; the query heads are the eight columns:
//     S^T[16 tokens, 8 heads] = K[16 tokens, dims] Q^T        O^T[16 dims, 8 heads] += V^T[16 dims, 16 tokens] P^T
// A code is already a bf16 number where it stands: bits 0-3 alone are c * 2^-133, bits 4-7 alone (the top one is the exponent's lowest bit) c * 2^-129, both exact, as
// bf16 numbers below 2^-125 are evenly spaced. So one AND makes two operands, and a shift by 8 the other two of a 16-bit unit. The powers of two go into the other
// operand, which is bf16 with all of its exponents to spare: the query's values are multiplied by a power of two per head, the weights by one that follows the values' scales.
// The offset of 7.5 levels is taken off in 32 bits: from the keys' products by the sum of the query's values, from the values' by a product with a row of equal codes that
// sums the weights. Scales multiply the products of a group of keys, and the weights of a group of values, in 32 bits. The place of codes in a page is
// such that a thread's registers are what it loads: no shuffle and no pass through shared memory. A thread's rows of S^T are the
// tokens 4 (r / 2) + r % 2 and two later (r = lane / 4), so that the columns it has to hold of V^T are four consecutive tokens.
//
// tcgen05 would want the unpacked keys and values written to shared or tensor memory first; the unpacking is what bounds the kernel, not the products (a third of
// mma.sync's rate at long contexts): 5 of a word's instructions are its unpacking, 65 of 125 million instructions of the case below run on the integer pipe.
//
// Measured (a graph of calls on states larger than L2): 32 sequences of 32768 tokens, 32 query and 8 KV heads of 128: 217 us, 5.57 TB/s, 0.85 of what a plain copy moves;
// 258 us back to back for seconds, at the board's power limit. 64 / 8 heads 242 us. 64 of 4000 67 us, 128 of 4000 113 us, 64 of 1280 27 us (two waves of CTAs), one of
// 131072 with 40 heads 45 us, one of 4000 9.1 us, 48 of 1024 with heads of 256 30 us. Short calls are a chain of latencies: length, page, keys, a step's products and softmax
// (some 0.8 us a step of a warp alone on its scheduler, however many steps are on their way), the join.
//
// The reference's counterpart is the paged attention behind vLLM's kv_cache_dtype (nemo_rl/models/generation/vllm/config.py).
#include "kv4.cuh"

#include <math.h>

namespace {
using namespace rlb;

constexpr int K4_WARPS = 4;
constexpr int K4_STEP = 32;      // tokens a warp takes at a time: twice the 16 of an instruction
constexpr int K4_CLUSTER = 8;    // CTAs of a cluster at most
constexpr int K4_FOLD = 16;      // steps between two corrections of the sums
constexpr float K4_SLACK = 8.f;  // how far (in powers of two) a score may pass the running maximum before the sums are rescaled: weights stay below 2^8
// Weights are held 2^lift times as large, so that their products with the largest of the values' scales seen so far start near 2^88. Above, 28 powers of two are left until the
// next change of the lift, and K4_SLACK: products stay below 2^125, of bf16's 2^128. Below, a product of 2^-9 is the least whose eight bits all count in 32 bits (a code's unit
// is 2^-133, the least number 2^-149): weight times scale may be 2^-97 of the largest scale, and by the lift's end of 92 2^-101 (no scale is below 2^-103). That end is there for
// the denominator: lifted weights of 2^27 tokens have a sum.
constexpr int K4_LIFT = 88, K4_ROOM = 28, K4_MOST = 92;

struct K4Params {
  const __nv_bfloat16* q;
  long long q_stride;
  const uint8_t* cache;
  long long num_blocks;
  const int* block_table;
  long long table_stride;
  int max_blocks;
  const int* seq_lens;
  int Hkv, G, chunks, block_size, window;
  float scale;
  int B, num_ctas, cluster;      // num_ctas: CTAs that share all tokens evenly, or 0: a cluster of `cluster` CTAs per (sequence, heads)
  float* part_o;        // [num_ctas][2] parts of 8 heads x D sums
  float2* part_ml;      // [num_ctas][2][8]
  int4* joins;          // [min(num_ctas, sequences x heads)]
  __nv_bfloat16* out;
  long long out_stride;
  int* status;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }      // e from -126 to 127
// Codes at nibble j of both halves of a word as two bf16 numbers: code * 2^-133 for even j, code * 2^-129 for odd j.
__device__ __forceinline__ uint32_t unpack2(uint32_t w, int j) { return w & (j & 1 ? 0x00f000f0u : 0x000f000fu); }
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 16 tokens' products of a group of 32 dimensions: wa, wb are the thread's words of its two tokens, q its pairs of the query.
__device__ __forceinline__ void score_group(float (&acc)[4], uint32_t wa, uint32_t wb, uint4 q) {
  mma_bf16(acc, unpack2(wa, 0), unpack2(wb, 0), unpack2(wa, 1), unpack2(wb, 1), q.x, q.y);
  wa >>= 8;
  wb >>= 8;
  mma_bf16(acc, unpack2(wa, 0), unpack2(wb, 0), unpack2(wa, 1), unpack2(wb, 1), q.z, q.w);
}
// 32 dimensions of 16 tokens' values added to the sums of a group: weights w0, w1.
__device__ __forceinline__ void add_group(float (&o0)[4], float (&o1)[4], uint32_t wa, uint32_t wb, uint32_t w0, uint32_t w1) {
  mma_bf16(o0, unpack2(wa, 0), unpack2(wa, 1), unpack2(wb, 0), unpack2(wb, 1), w0, w1);
  wa >>= 8;
  wb >>= 8;
  mma_bf16(o1, unpack2(wa, 0), unpack2(wa, 1), unpack2(wb, 0), unpack2(wb, 1), w0, w1);
}
// Two sums or products at once.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
// 2^e for e from -252 to 254, as two factors where one would not do.
__device__ __forceinline__ float times_pow2(float x, int e) {
  const int h = e >> 1;
  return x * pow2(h) * pow2(e - h);
}

// N words of shared memory at once; 16 bytes from global to shared memory, in the background.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* from, uint32_t (&w)[N]) {
  if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(from);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = reinterpret_cast<const uint4*>(from)[i / 4];
      w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
    }
  }
}
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ float2 ld_cluster2(uint32_t from) {      // of another CTA of the cluster
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(from) : "memory");
  return v;
}
// p + a * b, in one multiplication.
__device__ __forceinline__ const uint8_t* wide(const uint8_t* p, uint32_t a, uint32_t b) { return p + static_cast<unsigned long long>(a) * b; }
__device__ __forceinline__ float bf16_of(uint32_t word, int i) { return __uint_as_float(i & 1 ? word & 0xffff0000u : word << 16); }

// A warp's stage: twice 16 tokens of keys, values and scales. They are copied as they lie, 512 bytes by a warp's instruction (each lane the words that it uses would be four
// times as many requests for the values: 32 sequences of 32768 tokens 225 instead of 216 us), 32 bytes to one place. The places are such that neither the copies nor the lanes that read
// meet in a bank:
//   keys    words of a lane's token a at lane * 4 G, those of token b (two later) 4 D bytes behind
//   values  pair a of a lane (r, t) at 4 G (8 t + (r ^ 2 t)), pair b 4 D bytes behind
// but with a bit of the address turned where more than 128 bytes are read at once: for b with heads of 64, for the second 16 bytes of a lane with heads of 256.
template <int D>
struct K4Stage {
  static constexpr int KEYS = 0, VALUES = 8 * D, SCALES = 16 * D, HALF = 18 * D, BYTES = 2 * HALF;
  static constexpr int COUNT = D == 64 ? 4 : D == 128 ? 3 : 2;      // steps whose words are in a warp's shared memory or on their way
  // 16 bytes `k` * 512 + lane * 16 of 16 tokens' keys, or values, go to:
  __device__ static __forceinline__ int key_to(int lane, int k) {
    const int token = D == 64 ? lane >> 1 : D == 128 ? 8 * k + (lane >> 2) : 4 * k + (lane >> 3), r = (token >> 2) * 2 + (token & 1), b = token >> 1 & 1;
    if constexpr (D == 64) return b * 256 + ((r * 32 + (lane & 1) * 16) ^ (b * 64));
    if constexpr (D == 128) return b * 512 + (4 * r + (lane & 3)) * 16;
    return b * 1024 + (4 * r + (lane >> 1 & 3)) * 32 + ((lane ^ r) & 1) * 16;
  }
  __device__ static __forceinline__ int value_to(int lane, int k) {
    const int pair = D == 64 ? lane >> 2 : D == 128 ? 4 * k + (lane >> 3) : 2 * k + (lane >> 4), t = pair >> 1, b = pair & 1;
    if constexpr (D == 64) return b * 256 + (t >> 1) * 128 + ((((t & 1) * 4 + ((lane & 3) ^ (t & 2))) ^ (b * 4)) * 16);
    if constexpr (D == 128) return b * 512 + t * 128 + ((lane & 7) ^ (2 * t)) * 16;
    return b * 1024 + t * 256 + ((lane >> 1 & 7) ^ (2 * t)) * 32 + ((lane ^ (t >> 1)) & 1) * 16;
  }
  // where a lane's words of its token or pair b stand, groups from 4 q on
  __device__ static __forceinline__ int key_at(int lane, int b, int q) {
    if constexpr (D == 64) return b * 256 + ((lane * 8) ^ (b * 64));
    if constexpr (D == 128) return b * 512 + lane * 16;
    return b * 1024 + lane * 32 + (q ^ (lane >> 2 & 1)) * 16;
  }
  __device__ static __forceinline__ int value_at(int lane, int b, int q) {
    const int r = lane >> 2, t = lane & 3;
    if constexpr (D == 64) return b * 256 + (t >> 1) * 128 + ((((t & 1) * 4 + ((r >> 1) ^ (t & 2))) ^ (b * 4)) * 16) + (r & 1) * 8;
    if constexpr (D == 128) return b * 512 + t * 128 + (r ^ (2 * t)) * 16;
    return b * 1024 + t * 256 + (r ^ (2 * t)) * 32 + (q ^ (t >> 1)) * 16;
  }
};
// Shared memory: the warps' stages; after the token loop [warps][8 heads] rows of D + 4 sums (4 more, for the banks) and [8 heads][D] of the CTA.
template <int D>
constexpr int k4_smem() {
  constexpr int fifo = K4_WARPS * K4Stage<D>::COUNT * K4Stage<D>::BYTES, red = K4_WARPS * 8 * (D + 4) * 4 + 8 * D * 4;
  return fifo > red ? fifo : red;
}

// Takes the codes' offset off the sums: z (of two groups, in rows 0-7 and 8-15) is 15 * 2^-133 times the weights, 7.5 levels of what rows 0-7 of a tile count in, and 1/16 of that of rows 8-15.
template <int G>
__device__ __forceinline__ void fold(float (&o)[2 * G][4], float (&z)[G / 2][4]) {
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float w = z[g >> 1][(g & 1) * 2 + (j & 1)];
      o[2 * g][j] = fmaf(j < 2 ? -0.5f : -8.f, w, o[2 * g][j]);
      o[2 * g + 1][j] = fmaf(j < 2 ? -0.5f : -8.f, w, o[2 * g + 1][j]);
    }
  }
#pragma unroll
  for (int g = 0; g < G / 2; ++g) z[g][0] = z[g][1] = z[g][2] = z[g][3] = 0.f;
}

// Tokens of a sequence that the table has room for, the first visible one, and the steps from there on.
struct K4Span {
  int len, first, step0, steps;
};
__device__ __forceinline__ K4Span k4_span(const K4Params& p, int b) {
  K4Span s;
  const long long room = p.num_blocks ? static_cast<long long>(p.max_blocks) * p.block_size : 0;
  s.len = p.seq_lens[b];
  if (s.len > room) {      // more tokens than the table has pages: recorded, the rest is left out
    if (p.status) atomicCAS(p.status, 0, RLB_ERR_BAD_ARG);
    s.len = static_cast<int>(room);
  }
  s.len = max(s.len, 0);
  s.first = p.window > 0 ? max(0, s.len - p.window) : 0;
  s.step0 = s.first / K4_STEP;
  s.steps = max(1, s.len / K4_STEP + (s.len % K4_STEP != 0) - s.step0);      // (one for an empty sequence, whose output is written too)
  return s;
}

template <int D, bool PAIR>
__global__ void __launch_bounds__(K4_WARPS * 32, D == 64 ? 4 : D == 128 ? 3 : 2) kv4_decode_kernel(const K4Params p) {
  extern __shared__ __align__(128) uint8_t k4_smem_raw[];
  __shared__ float2 ml[K4_WARPS][8];      // of each warp and column: what its weights are relative to (a power of two), and their sum
  __shared__ float2 joined_ml[8];
  __shared__ int found[2], sums[K4_WARPS];
  __shared__ uint4 query[PAIR ? 2 : 1][D / 32][32];      // each lane's operands of a group (PAIR: with zeros in columns 4-7, and in columns 0-3); what its products start from
  __shared__ float2 offset[D / 32][32];
  using Stage = K4Stage<D>;
  using Page = Kv4Page<D>;
  constexpr int STAGES = Stage::COUNT, G = Page::G, W = G < 4 ? G : 4;      // groups of 32 dimensions; words of a load
  constexpr int NS = PAIR ? 1 : 2;                   // times 16 tokens of a step that a column stands for
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int all_heads = p.Hkv * p.chunks;
  pdl_sync();

  // Which steps are this CTA's: those of one (sequence, heads), or an even share [x, x_end) of all of them in the order (heads, sequence, step).
  int b, hc, at, left = 1;             // sequence, heads, step within the sequence, steps from there on
  uint32_t share = 0;
  if (p.num_ctas) {
    const int per = (p.B + K4_WARPS * 32 - 1) / (K4_WARPS * 32), b0 = min(p.B, static_cast<int>(threadIdx.x) * per), b1 = min(p.B, b0 + per);
    int mine = 0;
    for (int i = b0; i < b1; ++i) mine += k4_span(p, i).steps;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < K4_WARPS; ++w) {
      if (w < warp) upto += sums[w];
      all += sums[w];
    }
    const uint32_t total = static_cast<uint32_t>(all) * all_heads, x = blockIdx.x * (share = (total + p.num_ctas - 1) / p.num_ctas);
    left = x < total ? static_cast<int>(min(share, total - x)) : 0;
    hc = static_cast<int>(x / all);
    int rest = static_cast<int>(x - hc * all) - (upto - mine);
    if (left && rest >= 0 && rest < mine) {      // (one thread)
      int i = b0;
      for (int n; (n = k4_span(p, i).steps) <= rest; ++i) rest -= n;
      found[0] = i;
      found[1] = rest;
    }
    __syncthreads();
    if (!left) {
      if (threadIdx.x == 0 && p.B * all_heads > p.num_ctas) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    b = found[0];
    at = found[1];
  } else {
    b = blockIdx.z * gridDim.y + blockIdx.y;
    if (static_cast<uint32_t>(b) >= static_cast<uint32_t>(p.B)) return;      // (with the whole cluster)
    hc = blockIdx.x / p.cluster;
    at = 0;
  }
  bool opened = false;      // whether a sequence begins here that goes on in the next CTA

  for (;;) {
  const int kvh = hc / p.chunks, chunk = hc - kvh * p.chunks, heads = min(8, p.G - chunk * 8), head0 = kvh * p.G + chunk * 8;
  const int col_head = PAIR ? r & 3 : r;      // the query head of column r
  const K4Span span = k4_span(p, b);
  int count = span.steps;
  if (p.num_ctas) {
    count = min(span.steps - at, left);
  } else if (p.cluster > 1) {      // (the clusters stand in a row)
    const int rank = blockIdx.x - hc * p.cluster;
    at = static_cast<int>(static_cast<long long>(span.steps) * rank / p.cluster);
    count = static_cast<int>(static_cast<long long>(span.steps) * (rank + 1) / p.cluster) - at;
  }
  const int len = span.len, first = span.first, begin = span.step0 + at;
  uint4 qv[G];
  {
    const __nv_bfloat16* q = p.q + static_cast<long long>(b) * p.q_stride + static_cast<long long>(head0 + col_head) * D + 8 * t;
#pragma unroll
    for (int g = 0; g < G; ++g) qv[g] = col_head < heads ? *reinterpret_cast<const uint4*>(q + 32 * g) : make_uint4(0, 0, 0, 0);
  }
  // The warp's steps are begin + warp + 4 i. Each lane knows the page of one half of a step (j = 2 i + half) among 16 of them, and of one among the 16 after.
  const int* table = p.block_table + static_cast<long long>(b) * p.table_stride;
  const int pos0 = (begin + warp) * K4_STEP, n = len && count > warp ? (count - warp + K4_WARPS - 1) / K4_WARPS : 0;
  // (Entries behind the sequence's pages may hold anything; page 0 is read in their place, and in that of a wrong one, which is recorded.)
  auto place = [&](int j, int& off) -> int {
    const int pos = pos0 + (j >> 1) * (K4_WARPS * K4_STEP) + (j & 1) * 16, blk = static_cast<int>(static_cast<uint32_t>(pos) / static_cast<uint32_t>(p.block_size));
    off = pos - blk * p.block_size;
    return blk < p.max_blocks ? table[blk] : 0;
  };
  auto checked = [&](int j, int no) -> int {
    const bool mine = j < 2 * n && pos0 + (j >> 1) * (K4_WARPS * K4_STEP) + (j & 1) * 16 < len, good = static_cast<uint32_t>(no) < static_cast<uint32_t>(p.num_blocks);
    if (mine && !good && p.status) atomicCAS(p.status, 0, RLB_ERR_BAD_ARG);
    return (mine && good ? no : 0) * p.Hkv + kvh;
  };
  int off_now = 0, off_next = 0;
  int page_next = place(32 + lane, off_next), page_now = checked(lane, place(lane, off_now));
  const uint32_t fifo = smem_u32(k4_smem_raw) + warp * (STAGES * Stage::BYTES);
  const int tok = 4 * (r >> 1) + (r & 1);      // of 16; the thread's other row is two tokens later
  const uint8_t *key_base = p.cache + lane * 16, *value_base = key_base + Page::values_at(p.block_size), *scale_base = key_base + Page::scales_at(p.block_size);
  const uint32_t page_bytes = static_cast<uint32_t>(Page::bytes(p.block_size));
  auto request = [&](int i) {
    if (i < n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int src = (2 * i + h) & 31;
        const uint32_t off = __shfl_sync(0xffffffffu, off_now, src), no = __shfl_sync(0xffffffffu, page_now, src);
        const uint8_t* keys = wide(wide(key_base, no, page_bytes), off, D / 2);
        const uint8_t* values = wide(wide(value_base, no, page_bytes), off, D / 2);
        const uint32_t to = fifo + (i % STAGES) * Stage::BYTES + h * Stage::HALF;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) copy16(to + Stage::KEYS + Stage::key_to(lane, k), keys + k * 512);
#pragma unroll
        for (int k = 0; k < D / 64; ++k) copy16(to + Stage::VALUES + Stage::value_to(lane, k), values + k * 512);
        if (lane < D / 8) copy16(to + Stage::SCALES + lane * 16, wide(wide(scale_base, no, page_bytes), off, D / 8));
      }
      if ((i & 15) == 15) {      // (an entry is looked at 16 steps after it was asked for)
        page_now = checked(2 * i + 2 + lane, page_next);
        off_now = off_next;
        page_next = place(2 * i + 34 + lane, off_next);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) request(i);

  // The queries as the 8-column operand: pair j of group g is (dimension 32 g + 8 t + j, and four later) of a head, times 2^k with the head's largest value
  // in [2^119, 2^120) (a sum of 32 stays finite), and 1/16 of that where the codes count 16 times. Scores are compared before they are scaled: a negative scale turns the
  // query's sign. c[h]: from the products' unit to powers of two, of columns 2 t and 2 t + 1.
  // They stay in shared memory, for the registers' sake, with -7.5 times the sum of the group's values of columns 2 t and 2 t + 1 (a product with a row of codes 15, halved).
  float c[2], slack[2];
  {
    uint32_t big = 0u;
#pragma unroll
    for (int g = 0; g < G; ++g)
      big = __vmaxu2(__vmaxu2(big, __vmaxu2(qv[g].x & 0x7fff7fffu, qv[g].y & 0x7fff7fffu)), __vmaxu2(qv[g].z & 0x7fff7fffu, qv[g].w & 0x7fff7fffu));
    big = max(big & 0xffffu, big >> 16);
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const int k = 119 + 127 - static_cast<int>(big >> 7);      // -9 to 246: in two factors, the second also with the sign, and with 1/16
    const float half = pow2(k >> 1), rest = pow2(k - (k >> 1)) * (p.scale < 0.f ? -1.f : 1.f);
    const uint32_t by = pack_bf16x2(half, half), by_even = pack_bf16x2(rest, rest), by_odd = pack_bf16x2(rest * 0.0625f, rest * 0.0625f);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if ((g & (K4_WARPS - 1)) != warp) continue;      // (the warps take turns)
      const uint32_t w[4] = {__byte_perm(qv[g].x, qv[g].z, 0x5410), __byte_perm(qv[g].x, qv[g].z, 0x7632), __byte_perm(qv[g].y, qv[g].w, 0x5410), __byte_perm(qv[g].y, qv[g].w, 0x7632)};
      uint32_t qf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) qf[j] = mul_bf16x2(mul_bf16x2(w[j], by), j & 1 ? by_odd : by_even);
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      const uint4 all = make_uint4(qf[0], qf[1], qf[2], qf[3]), none = make_uint4(0u, 0u, 0u, 0u);
      score_group(acc, 0xffffffffu, 0xffffffffu, all);
      query[0][g][lane] = PAIR && r >= 4 ? none : all;
      if constexpr (PAIR) query[NS][g][lane] = r >= 4 ? all : none;
      offset[g][lane] = make_float2(-0.5f * acc[0], -0.5f * acc[1]);
    }
    // (never 0, so that -inf times it stays -inf; the slack is finite, so that any score passes -inf)
    const float unit = fminf(fmaxf(times_pow2(fabsf(p.scale) * 1.4426950408889634f, 133 - k), 0x1p-149f), 0x1p127f);
    c[0] = __shfl_sync(0xffffffffu, unit, 8 * t);
    c[1] = __shfl_sync(0xffffffffu, unit, 8 * t + 4);
    slack[0] = fminf(K4_SLACK / c[0], 0x1p127f);
    slack[1] = fminf(K4_SLACK / c[1], 0x1p127f);
  }
  __syncthreads();

  float o[2 * G][4], z[G / 2][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
  // limit: the largest scale, in bf16 bits in both halves, that the lift is good for.
  float lift = 0.f, ref[2] = {0.f, 0.f};      // ref: what is added to a score's power of two
  uint32_t limit = 0u;
#pragma unroll
  for (int i = 0; i < 2 * G; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
  for (int g = 0; g < G / 2; ++g) z[g][0] = z[g][1] = z[g][2] = z[g][3] = 0.f;

  for (int i = 0; i < n; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();      // every lane copied for the others; and has read the stage that is requested next
    request(i + STAGES - 1);
    const uint8_t* from = k4_smem_raw + (warp * STAGES + i % STAGES) * Stage::BYTES;
    float s[NS][4];
    uint32_t va[NS][G / 2], vb[NS][G / 2];      // the values' scales
#pragma unroll
    for (int h = 0; h < NS; ++h) {
      const uint8_t* mine = from + (PAIR ? t >> 1 : h) * Stage::HALF;      // (columns 0-3: the first 16 tokens, 4-7: the others)
      uint32_t sa[G], sb[G];
      load_words(mine + Stage::SCALES + Page::scale(tok, 0, 0), sa);
      load_words(mine + Stage::SCALES + Page::scale(tok + 2, 0, 0), sb);
      float2 lo = make_float2(0.f, 0.f), hi = lo;
#pragma unroll
      for (int g0 = 0; g0 < G; g0 += W) {
        uint32_t ka[W], kb[W], kc[W], kd[W];
        load_words(from + h * Stage::HALF + Stage::KEYS + Stage::key_at(lane, 0, g0 / 4), ka);
        load_words(from + h * Stage::HALF + Stage::KEYS + Stage::key_at(lane, 1, g0 / 4), kb);
        if constexpr (PAIR) {
          load_words(from + Stage::HALF + Stage::KEYS + Stage::key_at(lane, 0, g0 / 4), kc);
          load_words(from + Stage::HALF + Stage::KEYS + Stage::key_at(lane, 1, g0 / 4), kd);
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const int g = g0 + j;
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          score_group(acc, ka[j], kb[j], query[0][g][lane]);
          if constexpr (PAIR) score_group(acc, kc[j], kd[j], query[NS][g][lane]);
          const float2 start = offset[g][lane];
          const float fa = bf16_of(sa[g >> 1], g), fb = bf16_of(sb[g >> 1], g);
          lo = fma2(add2(make_float2(acc[0], acc[1]), start), make_float2(fa, fa), lo);
          hi = fma2(add2(make_float2(acc[2], acc[3]), start), make_float2(fb, fb), hi);
        }
      }
      s[h][0] = lo.x; s[h][1] = lo.y; s[h][2] = hi.x; s[h][3] = hi.y;
#pragma unroll
      for (int g = 0; g < G / 2; ++g) {
        va[h][g] = sa[G / 2 + g];
        vb[h][g] = sb[G / 2 + g];
      }
    }
    const int pos = pos0 + i * (K4_WARPS * K4_STEP);
    if (pos < first || pos + K4_STEP > len) {      // (a place that was never written, or by another sequence, may hold anything)
#pragma unroll
      for (int h = 0; h < NS; ++h) {
        const int token = pos + 16 * (PAIR ? t >> 1 : h) + tok;
        if (token < first || token >= len) {
          s[h][0] = s[h][1] = -INFINITY;
#pragma unroll
          for (int g = 0; g < G / 2; ++g) va[h][g] = 0u;
        }
        if (token + 2 < first || token + 2 >= len) {
          s[h][2] = s[h][3] = -INFINITY;
#pragma unroll
          for (int g = 0; g < G / 2; ++g) vb[h][g] = 0u;
        }
      }
    }
    // The running maximum moves only when a score passes it by K4_SLACK: weights are then at most 2^8, and any reference gives the same quotient.
    float m0 = fmaxf(s[0][0], s[0][2]), m1 = fmaxf(s[0][1], s[0][3]);
    if constexpr (!PAIR) {
      m0 = fmaxf(m0, fmaxf(s[NS - 1][0], s[NS - 1][2]));
      m1 = fmaxf(m1, fmaxf(s[NS - 1][1], s[NS - 1][3]));
    }
    uint32_t widest = limit;
#pragma unroll
    for (int h = 0; h < NS; ++h)
#pragma unroll
      for (int g = 0; g < G / 2; ++g) widest = __vmaxu2(widest, __vmaxu2(va[h][g], vb[h][g]));
    if (__any_sync(0xffffffffu, m0 > top[0] + slack[0] || m1 > top[1] + slack[1] || widest != limit)) {
      float f[2] = {1.f, 1.f}, rise = 1.f;
      uint32_t most = 0u, lost = 0u;      // the largest scale; groups with one that is not finite, which are NaN from here on (and count as zeros, for z's sake)
#pragma unroll
      for (int h = 0; h < NS; ++h)
#pragma unroll
        for (int g = 0; g < G / 2; ++g)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t& w = j ? vb[h][g] : va[h][g];
            if ((w & 0xffffu) >= 0x7f80u) {
              lost |= 1u << (2 * g);
              w &= 0xffff0000u;
            }
            if (w >> 16 >= 0x7f80u) {
              lost |= 2u << (2 * g);
              w &= 0xffffu;
            }
            most = max(most, max(w & 0xffffu, w >> 16));
          }
      most = __reduce_max_sync(0xffffffffu, most);
      lost = __reduce_or_sync(0xffffffffu, lost);
      if (lost) {
#pragma unroll
        for (int j = 0; j < 2 * G; ++j)
          if (lost >> (j >> 1) & 1u) o[j][0] = o[j][1] = o[j][2] = o[j][3] = __uint_as_float(0x7fc00000u);
      }
      if (most > (limit & 0xffffu)) {
        const int e = static_cast<int>(most >> 7) - 127;
        const int to = min(K4_MOST, K4_LIFT - e);      // -39 to 92
        rise = times_pow2(1.f, to - static_cast<int>(lift));      // 2^-131 at least, exactly: no token leaves the denominator when far larger values come
        lift = static_cast<float>(to);
        limit = static_cast<uint32_t>(min(254, max(1, e + K4_ROOM + 127))) << 7;
        limit |= limit << 16;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = h ? m1 : m0;
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        if (m > top[h]) {
          f[h] = exp2_fast((top[h] - m) * c[h]);      // (0 for the first)
          top[h] = m;
        }
        ref[h] = top[h] == -INFINITY ? 0.f : fmaf(-top[h], c[h], lift);
        sum[h] = sum[h] * f[h] * rise;
        f[h] *= rise;
#pragma unroll
        for (int j = 0; j < 2 * G; ++j) {
          o[j][h] *= f[h];
          o[j][h + 2] *= f[h];
        }
#pragma unroll
        for (int g = 0; g < G / 2; ++g) {
          z[g][h] *= f[h];
          z[g][h + 2] *= f[h];
        }
      }
    }
#pragma unroll
    for (int h = 0; h < NS; ++h) {
      const float2 pa = make_float2(exp2_fast(fmaf(s[h][0], c[0], ref[0])), exp2_fast(fmaf(s[h][1], c[1], ref[1])));
      const float2 pb = make_float2(exp2_fast(fmaf(s[h][2], c[0], ref[0])), exp2_fast(fmaf(s[h][3], c[1], ref[1])));
      sum[0] += pa.x + pb.x;
      sum[1] += pa.y + pb.y;
#pragma unroll
      for (int g0 = 0; g0 < G; g0 += W) {
        uint32_t wa[W], wb[W], wc[W], wd[W];
        load_words(from + h * Stage::HALF + Stage::VALUES + Stage::value_at(lane, 0, g0 / 4), wa);
        load_words(from + h * Stage::HALF + Stage::VALUES + Stage::value_at(lane, 1, g0 / 4), wb);
        if constexpr (PAIR) {
          load_words(from + Stage::HALF + Stage::VALUES + Stage::value_at(lane, 0, g0 / 4), wc);
          load_words(from + Stage::HALF + Stage::VALUES + Stage::value_at(lane, 1, g0 / 4), wd);
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const int g = g0 + j;
          const float fa = bf16_of(va[h][g >> 1], g), fb = bf16_of(vb[h][g >> 1], g);
          // weight * scale in 32 bits, rounded once to the operand's bf16: half a step, 2^-8 of each token's share at most, with either sign
          uint32_t w0 = transposed8x8(pack_bf16x2(pa.x * fa, pa.y * fa)), w1 = transposed8x8(pack_bf16x2(pb.x * fb, pb.y * fb));
          mma_bf16(z[g >> 1], g & 1 ? 0u : 0x000f000fu, g & 1 ? 0x000f000fu : 0u, g & 1 ? 0u : 0x000f000fu, g & 1 ? 0x000f000fu : 0u, w0, w1);
          if constexpr (PAIR) {      // columns 4-7 hold the weights of the other 16 tokens
            add_group(o[2 * g], o[2 * g + 1], wc[j], wd[j], r < 4 ? 0u : w0, r < 4 ? 0u : w1);
            w0 = r < 4 ? w0 : 0u;
            w1 = r < 4 ? w1 : 0u;
          }
          add_group(o[2 * g], o[2 * g + 1], wa[j], wb[j], w0, w1);
        }
      }
    }
    // The offset is taken off again and again: left until the end it would outgrow the sums, which are to keep their last bits.
    if (i % K4_FOLD == K4_FOLD - 1) fold<G>(o, z);
  }
  fold<G>(o, z);

  // The warps' parts (and, where four heads have two columns each, the columns') are brought to one reference and added: columns 2 t and 2 t + 1, dimensions
  // 32 g + 4 r .. + 3 of each lane. Tops are less the lift here, and lifts differ by up to 131. So a factor between parts, which 32 bits may
  // not hold, is applied as its root, twice: a part of tiny values keeps its share of the denominator beside one of huge values. Sums leave in 2^64 of the lifted values' unit, in
  // which alone they could pass the end of 32 bits.
  constexpr int PARTS = PAIR ? 2 * K4_WARPS : K4_WARPS;
  auto part_of = [&](int head, int i) -> float2 { return PAIR ? ml[i >> 1][head + 4 * (i & 1)] : ml[i][head]; };
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 4);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 8);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 16);
    top[h] = top[h] == -INFINITY ? -INFINITY : fmaf(top[h], c[h], -lift);
    if (r == 0) ml[warp][2 * t + h] = make_float2(top[h], sum[h]);
  }
  __syncthreads();      // (the stages' memory is used again, too)
  float* red = reinterpret_cast<float*>(k4_smem_raw);
  constexpr int ROW = D + 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int column = 2 * t + h, head = PAIR ? column & 3 : column;
    float m = part_of(head, 0).x;
#pragma unroll
    for (int i = 1; i < PARTS; ++i) m = fmaxf(m, part_of(head, i).x);
    // (a part without a finite score has no tokens, or NaN, which is to stay)
    const float root = top[h] == -INFINITY ? 1.f : exp2_fast(0.5f * (top[h] - m)), f = root * 0x1p34f, f0 = root * 0x1p35f, f1 = root * 0x1p31f;
#pragma unroll
    for (int g = 0; g < G; ++g)
      *reinterpret_cast<float4*>(red + (warp * 8 + column) * ROW + 32 * g + 4 * r) =
          make_float4(o[2 * g][h] * f * f0, o[2 * g][h + 2] * f * f1, o[2 * g + 1][h] * f * f0, o[2 * g + 1][h + 2] * f * f1);
  }
  __syncthreads();
  float* joined = red + K4_WARPS * 8 * ROW;
  for (int i = threadIdx.x; i < heads * (D / 4); i += K4_WARPS * 32) {
    const int head = i / (D / 4), d = i % (D / 4) * 4;
    float m = part_of(head, 0).x, l = 0.f;
#pragma unroll
    for (int w = 1; w < PARTS; ++w) m = fmaxf(m, part_of(head, w).x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < PARTS; ++w) {
      const float2 part = part_of(head, w);
      const float root = part.x == -INFINITY ? 1.f : exp2_fast(0.5f * (part.x - m));
      l += part.y * root * root;
      const float4 v = *reinterpret_cast<const float4*>(red + (PAIR ? (w >> 1) * 8 + head + 4 * (w & 1) : w * 8 + head) * ROW + d);
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    }
    if (p.cluster > 1) {
      *reinterpret_cast<float4*>(joined + head * D + d) = acc;
      if (d == 0) joined_ml[head] = make_float2(m, l);
    } else if (count == span.steps) {
      const float inv = l == 0.f ? 0.f : 0x1p64f / l;
      *reinterpret_cast<uint2*>(p.out + static_cast<long long>(b) * p.out_stride + static_cast<long long>(head0 + head) * D + d) =
          make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    } else {      // a part: of a sequence that began in an earlier CTA, or of one that begins here
      const long long part = static_cast<long long>(blockIdx.x) * 2 + (at == 0);
      *reinterpret_cast<float4*>(p.part_o + (part * 8 + head) * D + d) = acc;
      if (d == 0) p.part_ml[part * 8 + head] = make_float2(m, l);
    }
  }
  if (p.cluster > 1) {      // each CTA of the cluster writes its share of the output, from what all of them have
    cluster_sync();
    const uint32_t sums_at = smem_u32(joined), ml_at = smem_u32(joined_ml);
    for (int i = (blockIdx.x - hc * p.cluster) * (K4_WARPS * 32) + threadIdx.x; i < heads * (D / 4); i += p.cluster * (K4_WARPS * 32)) {
      const int head = i / (D / 4), d = i % (D / 4) * 4;
      float2 parts[K4_CLUSTER];
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int c = 0; c < K4_CLUSTER; ++c)
        if (c < p.cluster) {
          parts[c] = ld_cluster2(mapa_shared(ml_at + head * 8, c));
          m = fmaxf(m, parts[c].x);
        }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < K4_CLUSTER; ++c)
        if (c < p.cluster) {
          const float root = parts[c].x == -INFINITY ? 1.f : exp2_fast(0.5f * (parts[c].x - m));
          const uint32_t from = mapa_shared(sums_at + (head * D + d) * 4, c);
          const float2 u = ld_cluster2(from), v = ld_cluster2(from + 8);
          l = fmaf(parts[c].y * root, root, l);
          acc.x = fmaf(u.x * root, root, acc.x);
          acc.y = fmaf(u.y * root, root, acc.y);
          acc.z = fmaf(v.x * root, root, acc.z);
          acc.w = fmaf(v.y * root, root, acc.w);
        }
      const float inv = l == 0.f ? 0.f : 0x1p64f / l;
      *reinterpret_cast<uint2*>(p.out + static_cast<long long>(b) * p.out_stride + static_cast<long long>(head0 + head) * D + d) =
          make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    }
    cluster_sync();      // (the others may still read this CTA's sums)
  }
  if (!p.num_ctas) return;
  // A sequence that begins here is joined from this CTA's part and those of the CTAs up to the one that has its last step.
  if (at == 0) {
    int4 job = make_int4(-1, 0, 0, 0);
    if (count < span.steps) {
      opened = true;
      job = make_int4(static_cast<int>(blockIdx.x), static_cast<int>(((blockIdx.x + 1) * share - count + span.steps - 1) / share), b, hc);
    }
    if (threadIdx.x == 0) {
      if (p.B * all_heads <= p.num_ctas) p.joins[hc * p.B + b] = job;
      else if (opened) p.joins[blockIdx.x] = job;
    }
  }
  left -= count;
  if (!left) break;
  at = 0;
  if (++b == p.B) {
    b = 0;
    ++hc;
  }
  __syncthreads();      // the sums' memory becomes the stages' again
  }
  if (threadIdx.x == 0 && !opened && p.B * all_heads > p.num_ctas) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
}

// Joins the parts of the sequences that several CTAs shared. Few sequences: a CTA per sequence and head, whose eight warps take every eighth part. More than CTAs: at most
// one sequence begins in a CTA and ends in another, most of two parts; a CTA each, a warp per head.
template <int D, bool FEW>
__global__ void __launch_bounds__(256) kv4_join_kernel(const K4Params p) {
  __shared__ float4 red[FEW ? 8 : 1][D / 4];
  __shared__ float reds[8];
  constexpr int V = D / 128 > 0 ? D / 128 : 1, BY = FEW ? 8 : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = FEW ? blockIdx.y : warp;
  pdl_sync();
  const int4 job = p.joins[blockIdx.x];      // first and last CTA, sequence, heads
  const int kvh = job.w / p.chunks, chunk = job.w - kvh * p.chunks;
  if (job.x < 0 || head >= min(8, p.G - chunk * 8)) return;      // (FEW: the whole CTA)
  const int n = job.y - job.x + 1;
  auto part = [&](int i) { return (static_cast<long long>(job.x + i) * 2 + (i == 0)) * 8 + head; };
  float m = -INFINITY;
  for (int i = lane; i < n; i += 32) m = fmaxf(m, p.part_ml[part(i)].x);
  m = warp_max(m);
  float4 acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int i = FEW ? warp : 0; i < n; i += BY) {
    const long long from = part(i);
    const float2 w = p.part_ml[from];
    const float root = w.x == -INFINITY ? 1.f : exp2_fast(0.5f * (w.x - m));      // (a part without a finite score has no tokens, or NaN)
    l += w.y * root * root;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (lane + 32 * v < D / 4) {
        const float4 o = reinterpret_cast<const float4*>(p.part_o + from * D)[lane + 32 * v];
        acc[v].x = fmaf(o.x * root, root, acc[v].x);
        acc[v].y = fmaf(o.y * root, root, acc[v].y);
        acc[v].z = fmaf(o.z * root, root, acc[v].z);
        acc[v].w = fmaf(o.w * root, root, acc[v].w);
      }
  }
  if constexpr (FEW) {
    if (lane == 0) reds[warp] = l;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (lane + 32 * v < D / 4) red[warp][lane + 32 * v] = acc[v];
    __syncthreads();
    if (warp >= V) return;
    l = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) l += reds[q];
  }
  const float inv = l == 0.f ? 0.f : 0x1p64f / l;
  __nv_bfloat16* out = p.out + job.z * p.out_stride + static_cast<long long>(kvh * p.G + chunk * 8 + head) * D;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int d = lane + 32 * (FEW ? warp : v);
    if (d >= D / 4 || (FEW && v)) continue;
    float4 o = acc[v];
    if constexpr (FEW) {
      o = red[0][d];
#pragma unroll
      for (int q = 1; q < 8; ++q) {
        const float4 w = red[q][d];
        o.x += w.x; o.y += w.y; o.z += w.z; o.w += w.w;
      }
    }
    reinterpret_cast<uint2*>(out)[d] = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  }
}

// Shared memory of which an SM (227 KB) has room for `per_sm` CTAs, and no more.
constexpr int k4_room(int per_sm) { return (per_sm == 1 ? 116 : per_sm == 2 ? 77 : 58) * 1024; }

template <int D, bool PAIR>
int launch_decode(const K4Params& p, cudaStream_t stream) {
  static std::atomic<unsigned long long> ready{0};
  int dev = 0, sms = 0;
  cudaError_t e = kv4_device(dev, sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (!(ready.load() >> dev & 1)) {
    e = cudaFuncSetAttribute(kv4_decode_kernel<D, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, k4_room(1));
    if (e != cudaSuccess) return static_cast<int>(e);
    ready.fetch_or(1ull << dev);
  }
  const int all_heads = p.Hkv * p.chunks;
  cudaLaunchConfig_t cfg = {};
  constexpr int MOST = 65535;      // of a grid in its second and third direction
  cfg.gridDim = p.num_ctas ? dim3(p.num_ctas) : dim3(all_heads * p.cluster, p.B < MOST ? p.B : MOST, (p.B - 1) / MOST + 1);
  cfg.blockDim = dim3(K4_WARPS * 32);
  cfg.dynamicSmemBytes = k4_smem<D>();
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (p.cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = p.cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  if (rlb_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  // Fewer CTAs than the device holds are not spread evenly by themselves: some SMs get as many as they hold, others one, and the fullest takes the longest. So each asks for
  // so much shared memory that only as many fit an SM as have to (37 sequences of 2048 tokens, 8 heads of 128: 27.3 -> 22.0 us; 96 of 3001, 2 heads of 64 in
  // clusters of two: 21.7 -> 18.7), where that leaves the clusters their places: those of eight do not fill the SMs.
  const long long clusters = p.num_ctas ? p.num_ctas : static_cast<long long>(all_heads) * p.B;
  static std::atomic<int> held[KV4_DEVICES][K4_CLUSTER + 1][4];      // clusters that run at once with so many CTAs on an SM, plus one (0: not asked yet)
  for (int per_sm = 1; per_sm < 4 && k4_room(per_sm) > k4_smem<D>(); ++per_sm) {
    if (static_cast<long long>(sms) * per_sm < clusters * p.cluster) continue;
    int most = p.cluster == 1 ? sms * per_sm + 1 : held[dev][p.cluster][per_sm].load();
    cfg.dynamicSmemBytes = k4_room(per_sm);
    if (!most) {
      e = cudaOccupancyMaxActiveClusters(&most, kv4_decode_kernel<D, PAIR>, &cfg);
      if (e != cudaSuccess) return static_cast<int>(e);
      held[dev][p.cluster][per_sm].store(++most);
    }
    if (clusters < most) break;
    cfg.dynamicSmemBytes = k4_smem<D>();
  }
  e = cudaLaunchKernelEx(&cfg, kv4_decode_kernel<D, PAIR>, p);
  if (e != cudaSuccess || !p.num_ctas) return static_cast<int>(e);
  const long long segments = static_cast<long long>(p.B) * all_heads;
  if (segments <= p.num_ctas) rlb_launch_pdl(kv4_join_kernel<D, true>, dim3(static_cast<unsigned>(segments), p.G < 8 ? p.G : 8), dim3(256), 0, stream, p);
  else rlb_launch_pdl(kv4_join_kernel<D, false>, dim3(p.num_ctas), dim3(256), 0, stream, p);
  return static_cast<int>(cudaGetLastError());
}
}  // namespace

// q [B, >= Hq D] bf16, 16-byte aligned rows; block_table [B, max_blocks] int32; seq_lens [B]; out: 8-byte aligned rows. num_ctas: 0, for a cluster of `cluster` (1 to
// 8) CTAs per sequence and key/value head (and eight query heads), or CTAs that share all tokens evenly (cluster 1), with scratch part_o [num_ctas 16 D] and part_ml [num_ctas 36] fp32 (16-byte aligned).
RLB_API int rlb_kv4_paged_decode(const void* q, long long q_stride, const void* cache, long long num_blocks, const int* block_table, long long table_stride, int max_blocks,
                                 const int* seq_lens, int B, int Hq, int Hkv, int D, int block_size, int window, float scale, int cluster, int num_ctas, float* part_o, float* part_ml, void* out,
                                 long long out_stride, int* status, void* stream) {
  if ((D != 64 && D != 128 && D != 256) || Hkv < 1 || Hq < 1 || Hq % Hkv || block_size < 16 || block_size % 16 || block_size > KV4_MAX_BLOCK || window < 0) return -2;
  if (q_stride % 8 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache)) & 15)) return -2;
  if (out_stride % 4 || (reinterpret_cast<uintptr_t>(out) & 7)) return -2;
  if (B <= 0) return 0;
  const int group = Hq / Hkv, chunks = (group + 7) / 8;
  if (cluster < 1 || cluster > K4_CLUSTER || (num_ctas && cluster != 1)) return -3;
  if (num_ctas < 0 || (num_ctas && (!part_o || !part_ml || ((reinterpret_cast<uintptr_t>(part_o) | reinterpret_cast<uintptr_t>(part_ml)) & 15)))) return -3;
  const long long room = static_cast<long long>(max_blocks) * block_size, visible = window && window < room ? window : room, segments = static_cast<long long>(B) * Hkv * chunks;
  if (room > 0x7fff0000ll || segments > 0x7fffffffll || (num_ctas && segments * (visible / K4_STEP + 2) + num_ctas > 0x7fffffffll) ||
      static_cast<long long>(Hkv) * chunks * cluster > 0x7fffffffll || num_blocks * Hkv > 0x7fffffffll)
    return -4;
  const K4Params p{static_cast<const __nv_bfloat16*>(q), q_stride, static_cast<const uint8_t*>(cache), num_blocks, block_table, table_stride, max_blocks, seq_lens, Hkv, group, chunks,
                   block_size, window, scale, B, num_ctas, cluster, part_o, reinterpret_cast<float2*>(part_ml), reinterpret_cast<int4*>(part_ml + static_cast<long long>(num_ctas) * 32),
                   static_cast<__nv_bfloat16*>(out), out_stride, status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (group <= 4) return D == 64 ? launch_decode<64, true>(p, s) : D == 128 ? launch_decode<128, true>(p, s) : launch_decode<256, true>(p, s);
  return D == 64 ? launch_decode<64, false>(p, s) : D == 128 ? launch_decode<128, false>(p, s) : launch_decode<256, false>(p, s);
}
