// Writing and reading the 4-bit key/value cache of the generation engine (kv4.cuh has the format).
//
// Both kernels move every byte once and are bound by memory. Write: D / 16 threads take a head of a token, each eight dimensions of its lower half and the
// eight that these pair with in the rotation, so that the rotation needs no other thread; four neighbouring threads hold a group of 32 and find its largest
// magnitude with two shuffles. Read-back: four threads a head, each eight dimensions of every group, whose codes stand in one load.
//
// Measured (a graph of calls on states larger than L2): write of 15003 tokens of 32 + 2 * 8 heads of 128 62 us, 5.7 TB/s, 0.87 of what a plain copy moves (three quarters
// of the instruction slots are used); 64 tokens 2.7 us, one 2.5 us: a launch and two dependent loads. Read-back of 32771 tokens of 8 heads of 128 29.8 us, 5.8 TB/s, 0.88; 517 of 4 of 64 2.1 us.
//
// The reference reaches its quantised caches through vLLM's kv_cache_dtype (nemo_rl/models/generation/vllm/config.py).
#include "kv4.cuh"

#include <algorithm>

namespace {
using namespace rlb;

constexpr int KV4_READ_ROWS = 64;      // places a block of the read-back takes at most

// Sine and cosine of the product of a position and a frequency in 64 bits: at position p the rounding of the angle to 32 bits alone would be off by p
// / 2^25. Reduced to |r| <= pi/4 by a multiple of pi/2 that is subtracted in two parts (exact products by fma), then the Taylor series: the first term left out is
// below 3e-18.
__device__ __forceinline__ float2 turn(int position, float inv_freq) {
  const double a = static_cast<double>(position) * static_cast<double>(inv_freq);
  const double k = rint(a * 0.63661977236758134308);                       // 2 / pi
  double r = fma(-k, 1.5707963267948965580, a);                            // pi / 2 to 53 bits, and what that leaves
  r = fma(-k, 6.1232339957367660e-17, r);
  const double q = r * r;
  double s = 1.0 / 355687428096000.0, c = 1.0 / 20922789888000.0;          // 1 / 17!, 1 / 16!
  s = fma(s, q, -1.0 / 1307674368000.0);
  c = fma(c, q, -1.0 / 87178291200.0);
  s = fma(s, q, 1.0 / 6227020800.0);
  c = fma(c, q, 1.0 / 479001600.0);
  s = fma(s, q, -1.0 / 39916800.0);
  c = fma(c, q, -1.0 / 3628800.0);
  s = fma(s, q, 1.0 / 362880.0);
  c = fma(c, q, 1.0 / 40320.0);
  s = fma(s, q, -1.0 / 5040.0);
  c = fma(c, q, -1.0 / 720.0);
  s = fma(s, q, 1.0 / 120.0);
  c = fma(c, q, 1.0 / 24.0);
  s = fma(s, q, -1.0 / 6.0);
  c = fma(c, q, -0.5);
  s = fma(s * q, r, r);
  c = fma(c, q, 1.0);
  const long long n = static_cast<long long>(k);
  const float sf = static_cast<float>((n & 1) ? c : s), cf = static_cast<float>((n & 1) ? s : c);
  return make_float2(((n + 1) & 2) ? -cf : cf, (n & 2) ? -sf : sf);        // (cos, sin)
}

// Two pairs turned: products and sums rounded one by one (no fused multiply-add), so that codes are the same wherever the formula is computed in 32 bits.
__device__ __forceinline__ void turn2(uint32_t& lo, uint32_t& hi, float4 t) {
  const float2 a = unpack_bf16x2(lo), b = unpack_bf16x2(hi);
  lo = pack_bf16x2(__fsub_rn(__fmul_rn(a.x, t.x), __fmul_rn(b.x, t.y)), __fsub_rn(__fmul_rn(a.y, t.z), __fmul_rn(b.y, t.w)));
  hi = pack_bf16x2(__fadd_rn(__fmul_rn(b.x, t.x), __fmul_rn(a.x, t.y)), __fadd_rn(__fmul_rn(b.y, t.z), __fmul_rn(a.y, t.w)));
}

// Scale of the group whose 32 values four neighbouring threads hold (bf16 bits). The quotient by 7.5 rounded to bf16 is the same for a * (1 / 7.5)
// in 32 bits: 2 a 2^k / 15 is at least 2^-13 (relative) from the middle of two bf16 numbers.
__device__ __forceinline__ uint32_t group_scale(const uint4& v) {
  uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
  m = max(m & 0xffffu, m >> 16);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  if (m >= 0x7f80u) return 0x7fc0u;
  const float a = __uint_as_float(m << 16);
  if (a < 0x1p-100f) return 0u;
  return __bfloat16_as_ushort(__float2bfloat16_rn(a * (1.f / 7.5f)));
}

// Eight values' codes, the first in the low bits: floor(x / s) + 8, which lies in 0..15 by itself (|x / s| < 7.6), exactly. x and s have eight bits each, so that x / s is an
// integer or at least 2^-10 from every one but 0: the quotient by the reciprocal, off by less than 2^-19, plus 2^-12 has the right integer part, and below 0 it is kept below.
// Adding 1.5 * 2^23 rounds to an integer in the low bits; these bits are put together by multiplications, and what stands above them in each word comes off at the end.
__device__ __forceinline__ uint32_t codes8(const uint4& v, uint32_t scale) {
  if (scale == 0u || scale == 0x7fc0u) return 0x88888888u;
  const float inv = 1.f / __uint_as_float(scale << 16);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t out = 0u - 0x4b400000u * 0x11111111u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack_bf16x2(w[i]);
    float a = fmaf(f.x, inv, 7.5f + 0x1p-12f), b = fmaf(f.y, inv, 7.5f + 0x1p-12f);
    if (f.x < 0.f) a = fminf(a, 7.5f - 0x1p-12f);
    if (f.y < 0.f) b = fminf(b, 7.5f - 0x1p-12f);
    out += __float_as_uint(a + 12582912.f) * (1u << (8 * i)) + __float_as_uint(b + 12582912.f) * (16u << (8 * i));
  }
  return out;
}

// Page and place in it of a slot; page -1: none (negative, or outside the cache, which is recorded).
__device__ __forceinline__ int2 place_of(long long slot, int block_size, long long num_slots, int* status) {
  if (slot < 0) return make_int2(-1, 0);
  if (slot >= num_slots) {
    if (status) atomicCAS(status, 0, RLB_ERR_BAD_ARG);
    return make_int2(-1, 0);
  }
  const long long page = slot >> 32 ? slot / block_size : static_cast<long long>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(block_size));
  return make_int2(static_cast<int>(page), static_cast<int>(slot - page * block_size));
}

// Rotates the q and k heads of the fused rows in place and puts the rotated k and v into the cache. A block takes `rows` tokens and heads [h0, h0 +
// heads_per_block) of them, a row at a time: D / 16 threads a head, the next row's values on their way. The angles and the slots' places are worked out once per token.
template <int D>
__global__ void __launch_bounds__(256, 5) kv4_write_kernel(__nv_bfloat16* __restrict__ qkv, const int* __restrict__ pos, const float* __restrict__ inv_freq,
                                                        const long long* __restrict__ slots, uint8_t* __restrict__ cache, long long T, int Hq, int Hkv, int block_size,
                                                        long long row_stride, long long num_slots, int* status, int rows, int heads_per_block) {
  extern __shared__ __align__(16) float2 kv4_cs[];      // [rows][D / 2], then [rows] places
  using Page = Kv4Page<D>;
  constexpr int LPH = D / 16, HALF = D / 2, UP = D / 64;      // UP: the upper half's groups follow the lower half's
  int2* places = reinterpret_cast<int2*>(kv4_cs + rows * HALF);
  const long long t0 = static_cast<long long>(blockIdx.x) * rows;
  const int n = static_cast<int>(T - t0 < rows ? T - t0 : rows);
  const int h0 = blockIdx.y * heads_per_block, nh = min(heads_per_block, Hq + 2 * Hkv - h0);
  const int per_row = nh * LPH;
  pdl_sync();
  const int padded = (per_row + 31) / 32 * 32;      // (whole warps, for the shuffles)
  const long long next = row_stride / 8;
  uint4* p = nullptr;
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  auto first_row = [&](int w) {
    p = reinterpret_cast<uint4*>(qkv + t0 * row_stride + static_cast<long long>(h0) * D + (w / LPH) * D + w % LPH * 8);
    if (w < per_row) {
      lo = p[0];
      hi = p[HALF / 8];
    }
  };
  first_row(threadIdx.x);
  for (int i = threadIdx.x; i < n; i += blockDim.x) places[i] = place_of(slots[t0 + i], block_size, num_slots, status);
  if (h0 < Hq + Hkv)
    for (int i = threadIdx.x; i < n * HALF; i += blockDim.x) {      // (in the order in which a head's threads read 16 bytes each)
      const int j = i % HALF;
      kv4_cs[i - j + (j % 8 / 2 * LPH + j / 8) * 2 + j % 2] = turn(pos[t0 + i / HALF], inv_freq[j]);
    }
  __syncthreads();
  for (int w = threadIdx.x; w < padded; w += blockDim.x) {
    if (w != threadIdx.x) first_row(w);
    const int h = h0 + w / LPH, c = w % LPH;
    const bool live = w < per_row, value = h >= Hq + Hkv, held = live && h >= Hq;
    for (int r = 0; r < n; ++r, p += next) {
      uint4 lo_next = lo, hi_next = hi;
      if (live && r + 1 < n) {
        lo_next = p[next];
        hi_next = p[next + HALF / 8];
      }
      if (live && !value) {
        const float4* t = reinterpret_cast<const float4*>(kv4_cs + r * HALF) + c;
        turn2(lo.x, hi.x, t[0]);
        turn2(lo.y, hi.y, t[LPH]);
        turn2(lo.z, hi.z, t[2 * LPH]);
        turn2(lo.w, hi.w, t[3 * LPH]);
        p[0] = lo;
        p[HALF / 8] = hi;
      }
      const int2 place = places[r];
      if (__any_sync(0xffffffffu, held) && place.x >= 0) {      // (the place is the whole warp's)
        const uint32_t s_lo = group_scale(lo), s_hi = group_scale(hi);
        if (held) {
          const int t = c & 3, g = c >> 2, off = place.y;
          uint8_t* page = cache + (static_cast<long long>(place.x) * Hkv + (value ? h - Hq - Hkv : h - Hq)) * Page::bytes(block_size);
          const uint32_t c_lo = codes8(lo, s_lo), c_hi = codes8(hi, s_hi);
          if (value) {
            uint8_t* v = page + Page::values_at(block_size);
            *reinterpret_cast<uint16_t*>(v + Page::value_unit(off, 2 * t, g)) = static_cast<uint16_t>(c_lo);
            *reinterpret_cast<uint16_t*>(v + Page::value_unit(off, 2 * t + 1, g)) = static_cast<uint16_t>(c_lo >> 16);
            *reinterpret_cast<uint16_t*>(v + Page::value_unit(off, 2 * t, g + UP)) = static_cast<uint16_t>(c_hi);
            *reinterpret_cast<uint16_t*>(v + Page::value_unit(off, 2 * t + 1, g + UP)) = static_cast<uint16_t>(c_hi >> 16);
          } else {
            *reinterpret_cast<uint32_t*>(page + Page::key_word(off, t, g)) = c_lo;
            *reinterpret_cast<uint32_t*>(page + Page::key_word(off, t, g + UP)) = c_hi;
          }
          if (t == 0) {
            uint8_t* s = page + Page::scales_at(block_size);
            *reinterpret_cast<uint16_t*>(s + Page::scale(off, value, g)) = static_cast<uint16_t>(s_lo);
            *reinterpret_cast<uint16_t*>(s + Page::scale(off, value, g + UP)) = static_cast<uint16_t>(s_hi);
          }
        }
      }
      lo = lo_next;
      hi = hi_next;
    }
  }
}

template <int N>
__device__ __forceinline__ void words_of(const uint8_t* from, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(from);
  } else if constexpr (N == 2) {
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
// The numbers of codes at bits 3-6 of both halves times a scale: 16 + c as bf16, less 23.5, exactly; one rounding in the product.
__device__ __forceinline__ uint32_t values2(uint32_t codes, uint32_t scale) {
  uint32_t v;
  asm("{\n\t.reg .b32 x;\n\tsub.rn.bf16x2 x, %1, %2;\n\tmul.rn.bf16x2 %0, x, %3;\n\t}" : "=r"(v) : "r"((codes & 0x00780078u) | 0x41804180u), "r"(0x41bc41bcu), "r"(scale));
  return v;
}
// Eight values of a word (the first in the low bits) by their scale in both halves.
__device__ __forceinline__ uint4 values8(uint32_t codes, uint32_t scale) {
  const uint32_t a = values2(codes << 3, scale), b = values2(codes >> 1, scale), c = values2(codes >> 5, scale), d = values2(codes >> 9, scale);      // (0, 4), (1, 5), (2, 6), (3, 7)
  return make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x7632));
}

// Keys and values of places of the cache as bf16 rows [k | v]. out_rows: which row of `out` a place goes to (null: its own number). A negative slot gives zeros. A block
// takes `rows` places; four threads a head of each, with eight dimensions of every group.
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint8_t* __restrict__ cache, const long long* __restrict__ slots, const long long* __restrict__ out_rows,
                                                       __nv_bfloat16* __restrict__ out, long long n, long long out_stride, long long num_out, int Hkv, int block_size,
                                                       long long num_slots, int* status, int rows) {
  using Page = Kv4Page<D>;
  constexpr int G = Page::G;
  __shared__ int2 places[KV4_READ_ROWS];
  __shared__ long long targets[KV4_READ_ROWS];
  const long long first = static_cast<long long>(blockIdx.x) * rows;
  const int here = static_cast<int>(n - first < rows ? n - first : rows);
  pdl_sync();
  if (threadIdx.x < here) {
    const long long slot = slots[first + threadIdx.x];
    long long to = out_rows ? out_rows[first + threadIdx.x] : first + threadIdx.x;
    const int2 place = place_of(slot, block_size, num_slots, status);
    if (to < 0 || to >= num_out) {      // outside the output: recorded, nothing written
      if (status) atomicCAS(status, 0, RLB_ERR_BAD_ARG);
      to = -1;
    }
    places[threadIdx.x] = place;
    targets[threadIdx.x] = place.x < 0 && slot >= 0 ? -1 : to;
  }
  __syncthreads();
  const uint32_t per_row = 2 * Hkv * 4;
  for (uint32_t i = threadIdx.x; i < here * per_row; i += blockDim.x) {
    const uint32_t row = i / per_row, w = i - row * per_row;
    const int h = static_cast<int>(w >> 2), t = static_cast<int>(w & 3);
    const int2 place = places[row];
    const long long to = targets[row];
    if (to < 0) continue;
    uint4* p = reinterpret_cast<uint4*>(out + to * out_stride + static_cast<long long>(h) * D + t * 8);
    if (place.x < 0) {
#pragma unroll
      for (int g = 0; g < G; ++g) p[g * 4] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const bool value = h >= Hkv;
    const int off = place.y;
    const uint8_t* page = cache + (static_cast<long long>(place.x) * Hkv + (value ? h - Hkv : h)) * Page::bytes(block_size);
    uint32_t words[G], scales[G / 2];
    if (value) {      // units of two tokens lie side by side: both are read, one is taken
      uint32_t a[G], b[G];
      words_of(page + Page::values_at(block_size) + Page::value_unit(off & ~1, 2 * t, 0), a);
      words_of(page + Page::values_at(block_size) + Page::value_unit(off & ~1, 2 * t + 1, 0), b);
#pragma unroll
      for (int g = 0; g < G; ++g) words[g] = __byte_perm(a[g], b[g], off & 1 ? 0x7632 : 0x5410);
    } else {
      words_of(page + Page::key_word(off, t, 0), words);
    }
    words_of(page + Page::scales_at(block_size) + Page::scale(off, value, 0), scales);
#pragma unroll
    for (int g = 0; g < G; ++g) p[g * 4] = values8(words[g], __byte_perm(scales[g >> 1], 0u, g & 1 ? 0x3232 : 0x1010));
  }
}

template <int D>
int launch_write(void* qkv, const int* pos, const float* inv_freq, const long long* slots, void* cache, long long T, int Hq, int Hkv, int block_size, long long row_stride,
                 long long num_blocks, int* status, cudaStream_t stream) {
  const int heads = Hq + 2 * Hkv, per_head = D / 16;
  int dev = 0, sms = 0;
  const cudaError_t e = kv4_device(dev, sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  const bool many = T * heads * per_head > static_cast<long long>(sms) * 2048;      // more than the device holds threads: whole rows, some tokens a block (15003 tokens of 32 + 2 * 8 heads of 128, us with 2, 4, 8: 62, 64, 69; 32 + 2 * 4 of 64: 31, 29, 30; 16 + 2 * 8 of 256 with 1, 2, 4: 2500 tokens 20.0, 17.7, 18.7, 16000 104, 89, 87)
  const int rows = many ? (D == 64 ? 4 : 2) : 1, per_block = many ? heads : 128 / per_head;
  const int per_row = heads * per_head, times = (per_row + 255) / 256, threads = many ? ((per_row + times - 1) / times + 31) / 32 * 32 : 128;
  const dim3 grid(static_cast<unsigned>((T + rows - 1) / rows), static_cast<unsigned>((heads + per_block - 1) / per_block));
  rlb_launch_pdl(kv4_write_kernel<D>, grid, dim3(threads), rows * (D / 2 * sizeof(float2) + sizeof(int2)), stream, static_cast<__nv_bfloat16*>(qkv), pos, inv_freq, slots,
                 static_cast<uint8_t*>(cache), T, Hq, Hkv, block_size, row_stride, num_blocks * block_size, status, rows, per_block);
  return static_cast<int>(cudaGetLastError());
}

template <int D>
int launch_read(const void* cache, const long long* slots, const long long* out_rows, void* out, long long n, long long out_stride, long long num_out, int Hkv, int block_size,
                long long num_blocks, int* status, cudaStream_t stream) {
  const int per_row = 8 * Hkv, rows = std::max(1, std::min({KV4_READ_ROWS, 512 / per_row, static_cast<int>(std::min<long long>(n / 296 + 1, KV4_READ_ROWS))}));
  rlb_launch_pdl(kv4_read_kernel<D>, dim3(static_cast<unsigned>((n + rows - 1) / rows)), dim3(256), 0, stream, static_cast<const uint8_t*>(cache), slots, out_rows,
                 static_cast<__nv_bfloat16*>(out), n, out_stride, num_out, Hkv, block_size, num_blocks * block_size, status, rows);
  return static_cast<int>(cudaGetLastError());
}
bool bad_shape(int D, int Hkv, int block_size) { return (D != 64 && D != 128 && D != 256) || Hkv < 1 || block_size < 16 || block_size % 16 || block_size > KV4_MAX_BLOCK; }
}  // namespace

// qkv [T, (Hq + 2 Hkv) D] bf16, 16-byte aligned rows; pos [T]; inv_freq [D / 2]; slots [T] (block * block_size + offset; negative: rotate only); cache: see kv4.cuh.
RLB_API int rlb_rope_kv4_cache_write(void* qkv, const int* pos, const float* inv_freq, const long long* slots, void* cache, long long T, int Hq, int Hkv, int D, int block_size,
                                     long long row_stride, long long num_blocks, int* status, void* stream) {
  if (bad_shape(D, Hkv, block_size) || Hq < 0 || row_stride % 8 || ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(cache)) & 15)) return -2;
  if (T <= 0) return 0;
  if (T > 0x7fffffffll || num_blocks > 0x7fffffffll || (Hq + 2ll * Hkv) * (D / 16) / 128 + 1 > 65535) return -3;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = D == 64 ? launch_write<64> : D == 128 ? launch_write<128> : launch_write<256>;
  return launch(qkv, pos, inv_freq, slots, cache, T, Hq, Hkv, block_size, row_stride, num_blocks, status, s);
}

// out [num_out, >= 2 Hkv D] bf16, 16-byte aligned rows; slots [n]; out_rows [n] or null (row i goes to row i).
RLB_API int rlb_kv4_cache_read(const void* cache, const long long* slots, const long long* out_rows, void* out, long long n, long long out_stride, long long num_out, int Hkv, int D,
                               int block_size, long long num_blocks, int* status, void* stream) {
  if (bad_shape(D, Hkv, block_size) || out_stride % 8 || ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(cache)) & 15)) return -2;
  if (n <= 0) return 0;
  if (n > 0x7fffffffll || num_blocks > 0x7fffffffll || Hkv > (1 << 20)) return -3;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = D == 64 ? launch_read<64> : D == 128 ? launch_read<128> : launch_read<256>;
  return launch(cache, slots, out_rows, out, n, out_stride, num_out, Hkv, block_size, num_blocks, status, s);
}
