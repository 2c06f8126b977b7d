// Decode attention over the 4-bit key/value cache (kv4.cuh): one query token per sequence, softmax(scale q k^T) v over its cached tokens or the last
// `window` of them. One CTA of four warps per (sequence, key/value head and up to eight of its query heads, split of the tokens).
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
// tcgen05 would want the unpacked keys and values written to shared or tensor memory first; the unpacking is what bounds the kernel, not the products.
//
// The reference's counterpart is the paged attention behind vLLM's kv_cache_dtype (nemo_rl/models/generation/vllm/config.py).
#include "kv4.cuh"

#include <math.h>

#include <atomic>

namespace {
using namespace rlb;

constexpr int K4_WARPS = 4;
constexpr int K4_STEP = 16;      // tokens a warp takes at a time
constexpr int K4_STAGES = 4;     // steps whose words are in a warp's shared memory or on their way
constexpr int K4_FOLD = 16;      // steps between two corrections of the sums
constexpr float K4_SLACK = 8.f;  // how far (in powers of two) a score may pass the running maximum before the sums are rescaled: weights stay below 2^8

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
  int num_splits;
  float* part_o;
  float* part_ml;
  __nv_bfloat16* out;
  long long out_stride;
  int* status;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Codes at nibble j of both halves of a word as two bf16 numbers: code * 2^-133 for even j, code * 2^-129 for odd j.
__device__ __forceinline__ uint32_t unpack2(uint32_t w, int j) { return (j & 2 ? w >> 8 : w) & (j & 1 ? 0x00f000f0u : 0x000f000fu); }
// 2^e for e from -252 to 254, as two factors where one would not do.
__device__ __forceinline__ float times_pow2(float x, int e) {
  const int h = e >> 1;
  return x * __uint_as_float(static_cast<uint32_t>(h + 127) << 23) * __uint_as_float(static_cast<uint32_t>(e - h + 127) << 23);
}

// N words of shared memory at once; and from global to shared memory, in the background.
template <int N>
__device__ __forceinline__ void load_words(uint32_t from, uint32_t (&w)[N]) {
  if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(from));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(from + 4 * i));
  }
}
template <int N>
__device__ __forceinline__ void copy_words(uint32_t to, const uint8_t* from) {
  if constexpr (N == 2) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 4 * i), "l"(from + 4 * i) : "memory");
  }
}
__device__ __forceinline__ float bf16_of(uint32_t word, int i) { return __uint_as_float(i & 1 ? word & 0xffff0000u : word << 16); }

// A warp's stage: the words that each lane is going to use (its own copies, so that no other lane has to be waited for), and the scales of the 16 tokens.
template <int D>
struct K4Stage {
  static constexpr int PART = 32 * (D / 32) * 4;      // one word per lane and group
  static constexpr int KA = 0, KB = PART, VA = 2 * PART, VB = 3 * PART, SCALES = 4 * PART, BYTES = 4 * PART + 2 * D;
};
// Shared memory: the warps' stages; after the token loop [warps][8 heads][D] sums, then [warps][8][2] maximum and sum of the weights.
template <int D>
constexpr int k4_smem() {
  constexpr int fifo = K4_WARPS * K4_STAGES * K4Stage<D>::BYTES, red = K4_WARPS * 8 * (D + 2) * 4;
  return fifo > red ? fifo : red;
}

// Takes the codes' offset off the sums: z is 15 * 2^-133 times the weights, 7.5 levels of what rows 0-7 of a tile count in, and 1/16 of that of rows 8-15.
template <int G>
__device__ __forceinline__ void fold(float (&o)[2 * G][4], float (&z)[G][4]) {
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[2 * g][j] = fmaf(j < 2 ? -0.5f : -8.f, z[g][j & 1], o[2 * g][j]);
      o[2 * g + 1][j] = fmaf(j < 2 ? -0.5f : -8.f, z[g][j & 1], o[2 * g + 1][j]);
    }
    z[g][0] = z[g][1] = z[g][2] = z[g][3] = 0.f;
  }
}

template <int D>
__global__ void __launch_bounds__(K4_WARPS * 32, D <= 128 ? 4 : 2) kv4_decode_kernel(const K4Params p) {
  extern __shared__ __align__(128) uint8_t k4_smem_raw[];
  using Stage = K4Stage<D>;
  using Page = Kv4Page<D>;
  constexpr int G = Page::G;      // groups of 32 dimensions
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int b = blockIdx.z, kvh = blockIdx.y / p.chunks, chunk = blockIdx.y % p.chunks, split = blockIdx.x;
  const int heads = min(8, p.G - chunk * 8), head0 = kvh * p.G + chunk * 8;
  pdl_sync();

  int len = p.seq_lens[b];
  const long long room = p.num_blocks ? static_cast<long long>(p.max_blocks) * p.block_size : 0;
  if (len > room) {      // more tokens than the table has pages: recorded, the rest is left out
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, RLB_ERR_BAD_ARG);
    len = static_cast<int>(room);
  }
  len = max(len, 0);
  const int first = p.window > 0 ? max(0, len - p.window) : 0;
  const int step0 = first / K4_STEP, steps = len / K4_STEP + (len % K4_STEP != 0) - step0;
  const int begin = step0 + static_cast<int>(static_cast<long long>(steps) * split / p.num_splits);
  const int end = step0 + static_cast<int>(static_cast<long long>(steps) * (split + 1) / p.num_splits);

  // The queries as the 8-column operand: pair j of group g is (dimension 32 g + 8 t + j, and four later) of head r, times 2^k with the head's largest value
  // in [2^119, 2^120) (a sum of 32 stays finite), and 1/16 of that where the codes count 16 times. Scores are compared before they are scaled: a negative scale turns the
  // query's sign. c[h]: from the products' unit to powers of two, of heads 2 t and 2 t + 1.
  uint32_t qf[G][4];
  float start[G][2], c[2], slack[2];      // start: -7.5 * sum of the group's values
  {
    const __nv_bfloat16* q = p.q + static_cast<long long>(b) * p.q_stride + static_cast<long long>(head0 + r) * D + 8 * t;
    uint4 v[G];
    uint32_t big = 0u;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      v[g] = make_uint4(0, 0, 0, 0);
      if (r < heads) v[g] = *reinterpret_cast<const uint4*>(q + 32 * g);
      big = max(max(max(big, v[g].x & 0x7fffu), max(v[g].x >> 16 & 0x7fffu, v[g].y & 0x7fffu)), max(v[g].y >> 16 & 0x7fffu, v[g].z & 0x7fffu));
      big = max(max(big, v[g].z >> 16 & 0x7fffu), max(v[g].w & 0x7fffu, v[g].w >> 16 & 0x7fffu));
    }
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const int k = 119 + 127 - static_cast<int>(big >> 7);
    const float sign = p.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t w[4] = {v[g].x, v[g].y, v[g].z, v[g].w};
      float f[8], s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = unpack_bf16x2(w[i]);
        f[2 * i] = times_pow2(a.x * sign, k);
        f[2 * i + 1] = times_pow2(a.y * sign, k);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s += f[j] + f[4 + j];
        qf[g][j] = pack_bf16x2(f[j] * (j & 1 ? 0.0625f : 1.f), f[4 + j] * (j & 1 ? 0.0625f : 1.f));
      }
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      s = times_pow2(s * -7.5f, -133);
      start[g][0] = __shfl_sync(0xffffffffu, s, 8 * t);
      start[g][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
    }
    const float unit = fminf(fmaxf(times_pow2(fabsf(p.scale) * 1.4426950408889634f, 133 - k), 1e-30f), 1e30f);
    c[0] = __shfl_sync(0xffffffffu, unit, 8 * t);
    c[1] = __shfl_sync(0xffffffffu, unit, 8 * t + 4);
    slack[0] = K4_SLACK / c[0];
    slack[1] = K4_SLACK / c[1];
  }

  float o[2 * G][4], z[G][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
  // Weights are held 2^lift times as large, so that their products with the values' scales lie near 2^40 and keep clear of the ends of 32 bits (times 2^-133) and of
  // bf16. limit: the largest scale, in bf16 bits in both halves, for which that holds.
  float lift = 0.f;
  uint32_t limit = 0u;
#pragma unroll
  for (int i = 0; i < 2 * G; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
  for (int g = 0; g < G; ++g) z[g][0] = z[g][1] = z[g][2] = z[g][3] = 0.f;

  // The warp's steps are begin + warp + 4 i. Each lane knows the page of one of 32 of them, and of one of the 32 after.
  const int* table = p.block_table + static_cast<long long>(b) * p.table_stride;
  const int n = end - begin > warp ? (end - begin - warp + K4_WARPS - 1) / K4_WARPS : 0;
  auto page_of = [&](int i, int& off) -> int {
    if (i >= n) return 0;
    const int pos0 = (begin + warp + i * K4_WARPS) * K4_STEP, blk = pos0 / p.block_size;
    off = pos0 - blk * p.block_size;
    int no = table[blk];
    if (no < 0 || no >= p.num_blocks) {      // outside the cache: recorded, and page 0 read in its place
      if (p.status) atomicCAS(p.status, 0, RLB_ERR_BAD_ARG);
      no = 0;
    }
    return no;
  };
  int off_now = 0, off_next = 0;
  int page_now = page_of(lane, off_now), page_next = page_of(32 + lane, off_next);
  const uint32_t fifo = smem_u32(k4_smem_raw) + warp * (K4_STAGES * Stage::BYTES);
  const int tok = 4 * (r >> 1) + (r & 1);      // of a step; the thread's other row is two tokens later
  auto request = [&](int i) {
    if (i < n) {
      const int src = i & 31;
      const int off = __shfl_sync(0xffffffffu, off_now, src);
      const uint8_t* page = p.cache + (static_cast<long long>(__shfl_sync(0xffffffffu, page_now, src)) * p.Hkv + kvh) * Page::bytes(p.block_size);
      const uint32_t to = fifo + (i % K4_STAGES) * Stage::BYTES;
      const uint8_t* keys = page + Page::key_word(off + tok, t, 0);
      const uint8_t* values = page + Page::values_at(p.block_size) + Page::value_unit(off + 4 * t, r, 0);
      copy_words<G>(to + Stage::KA + lane * (G * 4), keys);
      copy_words<G>(to + Stage::KB + lane * (G * 4), keys + D);               // two tokens of keys
      copy_words<G>(to + Stage::VA + lane * (G * 4), values);
      copy_words<G>(to + Stage::VB + lane * (G * 4), values + D);             // one pair of tokens of values
      if (lane < D / 8) copy_words<4>(to + Stage::SCALES + lane * 16, page + Page::scales_at(p.block_size) + Page::scale(off, 0, 0) + lane * 16);
      if (src == 31) {
        page_now = page_next;
        off_now = off_next;
        page_next = page_of(i + 33 + lane, off_next);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < K4_STAGES - 1; ++i) request(i);

  for (int i = 0; i < n; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(K4_STAGES - 2) : "memory");
    __syncwarp();      // the scales were copied by other lanes; and every lane has read the stage that is requested next
    const uint32_t from = fifo + (i % K4_STAGES) * Stage::BYTES;
    uint32_t ka[G], kb[G], va[G], vb[G], sa[G], sb[G];      // sa, sb: scales of keys, then of values
    load_words(from + Stage::KA + lane * (G * 4), ka);
    load_words(from + Stage::KB + lane * (G * 4), kb);
    load_words(from + Stage::SCALES + Page::scale(tok, 0, 0), sa);
    load_words(from + Stage::SCALES + Page::scale(tok + 2, 0, 0), sb);
    load_words(from + Stage::VA + lane * (G * 4), va);
    load_words(from + Stage::VB + lane * (G * 4), vb);
    request(i + K4_STAGES - 1);

    const int pos0 = (begin + warp + i * K4_WARPS) * K4_STEP;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      mma_bf16(acc, unpack2(ka[g], 0), unpack2(kb[g], 0), unpack2(ka[g], 1), unpack2(kb[g], 1), qf[g][0], qf[g][1]);
      mma_bf16(acc, unpack2(ka[g], 2), unpack2(kb[g], 2), unpack2(ka[g], 3), unpack2(kb[g], 3), qf[g][2], qf[g][3]);
      const float fa = bf16_of(sa[g >> 1], g), fb = bf16_of(sb[g >> 1], g);
      s[0] = fmaf(acc[0] + start[g][0], fa, s[0]);
      s[1] = fmaf(acc[1] + start[g][1], fa, s[1]);
      s[2] = fmaf(acc[2] + start[g][0], fb, s[2]);
      s[3] = fmaf(acc[3] + start[g][1], fb, s[3]);
    }
    const bool edge = pos0 < first || pos0 + K4_STEP > len;
    const bool live_a = pos0 + tok >= first && pos0 + tok < len, live_b = pos0 + tok + 2 >= first && pos0 + tok + 2 < len;
    if (edge) {      // (a place that was never written, or by another sequence, may hold anything)
      if (!live_a) s[0] = s[1] = -INFINITY;
      if (!live_b) s[2] = s[3] = -INFINITY;
#pragma unroll
      for (int g = G / 2; g < G; ++g) {      // (the values' scales)
        if (!live_a) sa[g] = 0u;
        if (!live_b) sb[g] = 0u;
      }
    }
    // The running maximum moves only when a score passes it by K4_SLACK: weights are then at most 2^8, and any reference gives the same quotient.
    uint32_t widest = limit;
#pragma unroll
    for (int g = G / 2; g < G; ++g) widest = __vmaxu2(widest, __vmaxu2(sa[g], sb[g]));
    if (__any_sync(0xffffffffu, fmaxf(s[0], s[2]) > top[0] + slack[0] || fmaxf(s[1], s[3]) > top[1] + slack[1] || widest != limit)) {
      float f[2] = {1.f, 1.f};
      uint32_t wide = 0u;      // the largest finite scale
#pragma unroll
      for (int g = G / 2; g < G; ++g) {
        const uint32_t w[4] = {sa[g] & 0xffffu, sa[g] >> 16, sb[g] & 0xffffu, sb[g] >> 16};
#pragma unroll
        for (int j = 0; j < 4; ++j) wide = max(wide, w[j] < 0x7f80u ? w[j] : 0u);
      }
      wide = __reduce_max_sync(0xffffffffu, wide);
      if (wide > (limit & 0xffffu)) {
        const int e = static_cast<int>(wide >> 7) - 127;
        const float to = static_cast<float>(max(-100, min(96, 40 - e)));
        f[0] = f[1] = exp2_fast(to - lift);
        lift = to;
        limit = static_cast<uint32_t>(min(254, max(1, e + 40 + 127))) << 7;
        limit |= limit << 16;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float m = fmaxf(s[h], s[h + 2]);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        if (m > top[h]) {
          f[h] *= exp2_fast((top[h] - m) * c[h]);      // (0 for the first)
          top[h] = m;
        }
        sum[h] *= f[h];
#pragma unroll
        for (int j = 0; j < 2 * G; ++j) {
          o[j][h] *= f[h];
          o[j][h + 2] *= f[h];
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          z[g][h] *= f[h];
          z[g][h + 2] *= f[h];
        }
      }
    }
    const float ref0 = top[0] == -INFINITY ? 0.f : fmaf(-top[0], c[0], lift), ref1 = top[1] == -INFINITY ? 0.f : fmaf(-top[1], c[1], lift);
    const float p0 = exp2_fast(fmaf(s[0], c[0], ref0)), p1 = exp2_fast(fmaf(s[1], c[1], ref1)), p2 = exp2_fast(fmaf(s[2], c[0], ref0)), p3 = exp2_fast(fmaf(s[3], c[1], ref1));
    sum[0] += p0 + p2;
    sum[1] += p1 + p3;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float fa = bf16_of(sa[(G + g) >> 1], G + g), fb = bf16_of(sb[(G + g) >> 1], G + g);
      // weight * scale in 32 bits, rounded once to the operand's bf16: half a step, 2^-8 of each token's share at most, with either sign
      const uint32_t w0 = transposed8x8(pack_bf16x2(p0 * fa, p1 * fa)), w1 = transposed8x8(pack_bf16x2(p2 * fb, p3 * fb));
      mma_bf16(o[2 * g], unpack2(va[g], 0), unpack2(va[g], 1), unpack2(vb[g], 0), unpack2(vb[g], 1), w0, w1);
      mma_bf16(o[2 * g + 1], unpack2(va[g], 2), unpack2(va[g], 3), unpack2(vb[g], 2), unpack2(vb[g], 3), w0, w1);
      mma_bf16(z[g], 0x000f000fu, 0x000f000fu, 0x000f000fu, 0x000f000fu, w0, w1);
    }
    // The offset is taken off again and again: left until the end it would outgrow the sums, which are to keep their last bits.
    if (i % K4_FOLD == K4_FOLD - 1) fold(o, z);
  }
  fold(o, z);

  // the warps' parts: heads 2 t and 2 t + 1, dimensions 32 g + 4 r .. + 3
  __syncthreads();      // the FIFOs' memory is used again
  float* k4_red = reinterpret_cast<float*>(k4_smem_raw);
  float* red_ml = k4_red + K4_WARPS * 8 * D;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float l = sum[h];
    l += __shfl_xor_sync(0xffffffffu, l, 4);
    l += __shfl_xor_sync(0xffffffffu, l, 8);
    l += __shfl_xor_sync(0xffffffffu, l, 16);
    const int head = 2 * t + h;
    if (r == 0) {
      red_ml[(warp * 8 + head) * 2] = top[h] == -INFINITY ? -INFINITY : fmaf(top[h], c[h], -lift);      // what the weights are relative to
      red_ml[(warp * 8 + head) * 2 + 1] = l;
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
      *reinterpret_cast<float4*>(k4_red + (warp * 8 + head) * D + 32 * g + 4 * r) =
          make_float4(times_pow2(o[2 * g][h], 133), times_pow2(o[2 * g][h + 2], 129), times_pow2(o[2 * g + 1][h], 133), times_pow2(o[2 * g + 1][h + 2], 129));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += blockDim.x) {
    const int head = i / D, d = i - head * D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < K4_WARPS; ++w) m = fmaxf(m, red_ml[(w * 8 + head) * 2]);
    float l = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < K4_WARPS; ++w) {
      const float mw = red_ml[(w * 8 + head) * 2], f = mw == -INFINITY ? 0.f : exp2_fast(mw - m);
      const float lw = red_ml[(w * 8 + head) * 2 + 1], ow = k4_red[(w * 8 + head) * D + d];
      l += mw == -INFINITY ? lw : lw * f;      // (a part without a finite score: no tokens, or NaN)
      acc += mw == -INFINITY ? ow : ow * f;
    }
    if (p.num_splits == 1) {
      p.out[static_cast<long long>(b) * p.out_stride + static_cast<long long>(head0 + head) * D + d] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
    } else {
      const long long at = (static_cast<long long>(b) * p.Hkv * p.G + head0 + head) * p.num_splits + split;
      p.part_o[at * D + d] = acc;
      if (d == 0) {
        p.part_ml[at * 2] = m;
        p.part_ml[at * 2 + 1] = l;
      }
    }
  }
}

// Joins the splits: one CTA per (sequence, query head), a thread per dimension.
template <int D>
__global__ void __launch_bounds__(D) kv4_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, __nv_bfloat16* __restrict__ out, long long out_stride, int Hq,
                                                     int num_splits) {
  pdl_sync();
  const long long at = (static_cast<long long>(blockIdx.y) * Hq + blockIdx.x) * num_splits;
  float m = -INFINITY;
  for (int i = 0; i < num_splits; ++i) m = fmaxf(m, part_ml[(at + i) * 2]);
  float l = 0.f, acc = 0.f;
  for (int i = 0; i < num_splits; ++i) {
    const float mi = part_ml[(at + i) * 2], f = mi == -INFINITY ? 1.f : exp2_fast(mi - m);
    l += part_ml[(at + i) * 2 + 1] * f;
    acc += part_o[(at + i) * D + threadIdx.x] * f;
  }
  out[blockIdx.y * out_stride + static_cast<long long>(blockIdx.x) * D + threadIdx.x] = __float2bfloat16_rn(l == 0.f ? 0.f : acc / l);
}

template <int D>
int launch_decode(const K4Params& p, int B, cudaStream_t stream) {
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (!(ready.load() >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(kv4_decode_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, k4_smem<D>());
    if (e != cudaSuccess) return static_cast<int>(e);
    ready.fetch_or(1ull << (dev & 63));
  }
  rlb_launch_pdl(kv4_decode_kernel<D>, dim3(p.num_splits, p.Hkv * p.chunks, B), dim3(K4_WARPS * 32), k4_smem<D>(), stream, p);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.num_splits == 1) return static_cast<int>(e);
  rlb_launch_pdl(kv4_join_kernel<D>, dim3(p.Hkv * p.G, B), dim3(D), 0, stream, p.part_o, p.part_ml, p.out, p.out_stride, p.Hkv * p.G, p.num_splits);
  return static_cast<int>(cudaGetLastError());
}
}  // namespace

// q [B, >= Hq D] bf16, 16-byte aligned rows; block_table [B, max_blocks] int32; seq_lens [B]; part_o [B Hq splits D] and part_ml [B Hq splits 2] fp32 with more than one split.
RLB_API int rlb_kv4_paged_decode(const void* q, long long q_stride, const void* cache, long long num_blocks, const int* block_table, long long table_stride, int max_blocks,
                                 const int* seq_lens, int B, int Hq, int Hkv, int D, int block_size, int window, float scale, int num_splits, float* part_o, float* part_ml, void* out,
                                 long long out_stride, int* status, void* stream) {
  if ((D != 64 && D != 128 && D != 256) || Hkv < 1 || Hq < 1 || Hq % Hkv || block_size < 16 || block_size % 16 || block_size > KV4_MAX_BLOCK || window < 0) return -2;
  if (q_stride % 8 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache)) & 15)) return -2;
  if (B <= 0) return 0;
  if (num_splits < 1 || (num_splits > 1 && (!part_o || !part_ml))) return -3;
  const int group = Hq / Hkv, chunks = (group + 7) / 8;
  if (B > 65535 || Hkv * chunks > 65535 || (num_splits > 1 && B > 65535)) return -4;
  const K4Params p{static_cast<const __nv_bfloat16*>(q), q_stride, static_cast<const uint8_t*>(cache), num_blocks, block_table, table_stride, max_blocks, seq_lens, Hkv, group, chunks,
                   block_size, window, scale, num_splits, part_o, part_ml, static_cast<__nv_bfloat16*>(out), out_stride, status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return D == 64 ? launch_decode<64>(p, B, s) : D == 128 ? launch_decode<128>(p, B, s) : launch_decode<256>(p, B, s);
}
