// Writing and reading the 4-bit key/value cache of the generation engine (kv4.cuh has the format).
//
// Both kernels move every byte once and are bound by memory: D / 16 threads take a head of a token, each eight dimensions of its lower half and the
// eight that these pair with in the rotation, so that neither the rotation nor the unpacking needs another thread; four neighbouring threads hold
// a group of 32 and find its largest magnitude with two shuffles.
//
// The reference reaches its quantised caches through vLLM's kv_cache_dtype (nemo_rl/models/generation/vllm/config.py).
#include "kv4.cuh"

namespace {
using namespace rlb;

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

// floor(x / s) + 8 in 0..15, exactly: the quotient by the reciprocal is off by one at most, and the multiples of s that x lies between are exact in
// 32 bits (4 bits times 8).
__device__ __forceinline__ uint32_t code4(float x, float s, float inv) {
  float t = floorf(x * inv);
  t = __fmul_rn(t, s) > x ? t - 1.f : __fmul_rn(t + 1.f, s) <= x ? t + 1.f : t;
  return static_cast<uint32_t>(fminf(fmaxf(t + 8.f, 0.f), 15.f));
}
// Eight values' codes, the first in the low bits.
__device__ __forceinline__ uint32_t codes8(const uint4& v, uint32_t scale) {
  if (scale == 0u || scale == 0x7fc0u) return 0x88888888u;
  const float s = __uint_as_float(scale << 16), inv = 1.f / s;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack_bf16x2(w[i]);
    out |= code4(f.x, s, inv) << (8 * i) | code4(f.y, s, inv) << (8 * i + 4);
  }
  return out;
}

// Rotates the q and k heads of the fused rows in place and puts the rotated k and v into the cache. A block takes `rows` tokens and heads [h0, h0 +
// heads_per_block) of them; their angles are computed once.
template <int D>
__global__ void __launch_bounds__(256) kv4_write_kernel(__nv_bfloat16* __restrict__ qkv, const int* __restrict__ pos, const float* __restrict__ inv_freq,
                                                        const long long* __restrict__ slots, uint8_t* __restrict__ cache, long long T, int Hq, int Hkv, int block_size,
                                                        long long row_stride, long long num_slots, int* status, int rows, int heads_per_block) {
  extern __shared__ __align__(16) float2 kv4_cs[];
  using Page = Kv4Page<D>;
  constexpr int LPH = D / 16, HALF = D / 2;
  const long long t0 = static_cast<long long>(blockIdx.x) * rows;
  const int n = static_cast<int>(T - t0 < rows ? T - t0 : rows);
  const int h0 = blockIdx.y * heads_per_block, total_heads = Hq + 2 * Hkv;
  const int nh = min(heads_per_block, total_heads - h0);
  pdl_sync();
  if (h0 < Hq + Hkv) {
    for (int i = threadIdx.x; i < n * HALF; i += blockDim.x) kv4_cs[i] = turn(pos[t0 + i / HALF], inv_freq[i % HALF]);
  }
  __syncthreads();
  const int per_row = nh * LPH, total = n * per_row, lane = threadIdx.x & 31;
  for (int base = threadIdx.x - lane; base < total; base += blockDim.x) {      // (whole warps, for the shuffles)
    const int i = base + lane;
    const bool live = i < total;
    const int r = live ? i / per_row : 0, w = live ? i - r * per_row : 0, h = h0 + w / LPH, c = w % LPH;
    uint4* p = reinterpret_cast<uint4*>(qkv + (t0 + r) * row_stride + static_cast<long long>(h) * D + c * 8);
    const long long slot = live && h >= Hq ? slots[t0 + r] : -1;
    const bool store = slot >= 0 && slot < num_slots;
    if (slot >= num_slots && status && c == 0) atomicCAS(status, 0, RLB_ERR_BAD_ARG);      // outside the cache: recorded, rotated in place, not written
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    if (live && (h < Hq + Hkv || store)) {
      lo = p[0];
      hi = p[HALF / 8];
    }
    if (live && h < Hq + Hkv) {
      const float4* t = reinterpret_cast<const float4*>(kv4_cs + r * HALF + c * 8);
      turn2(lo.x, hi.x, t[0]);
      turn2(lo.y, hi.y, t[1]);
      turn2(lo.z, hi.z, t[2]);
      turn2(lo.w, hi.w, t[3]);
      p[0] = lo;
      p[HALF / 8] = hi;
    }
    if (!__any_sync(0xffffffffu, store)) continue;
    const uint32_t s_lo = group_scale(lo), s_hi = group_scale(hi);
    if (!store) continue;
    const bool value = h >= Hq + Hkv;
    const int head = value ? h - Hq - Hkv : h - Hq;
    const long long blk = slot / block_size;
    const int off = static_cast<int>(slot - blk * block_size), t = c & 3, g = c >> 2;
    uint8_t* page = cache + (blk * Hkv + head) * Page::bytes(block_size);
    const uint32_t c_lo = codes8(lo, s_lo), c_hi = codes8(hi, s_hi);
    constexpr int UP = D / 64;      // the upper half's groups follow the lower half's
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

__device__ __forceinline__ uint4 values8(uint32_t codes, uint32_t scale) {
  const float s = __uint_as_float(scale << 16);
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out[i] = pack_bf16x2((static_cast<float>(codes >> (8 * i) & 15u) - 7.5f) * s, (static_cast<float>(codes >> (8 * i + 4) & 15u) - 7.5f) * s);
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// Keys and values of places of the cache as bf16 rows [k | v]. out_rows: which row of `out` a place goes to (null: its own number). A negative slot gives zeros.
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint8_t* __restrict__ cache, const long long* __restrict__ slots, const long long* __restrict__ out_rows,
                                                       __nv_bfloat16* __restrict__ out, long long n, long long out_stride, long long num_out, int Hkv, int block_size,
                                                       long long num_slots, int* status) {
  using Page = Kv4Page<D>;
  constexpr int LPH = D / 16, UP = D / 64;
  pdl_sync();
  const int per_row = 2 * Hkv * LPH;
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long row = i / per_row;
  if (row >= n) return;
  const int w = static_cast<int>(i - row * per_row), h = w / LPH, c = w % LPH, t = c & 3, g = c >> 2;
  const long long to = out_rows ? out_rows[row] : row;
  const long long slot = slots[row];
  if (to < 0 || to >= num_out || slot >= num_slots) {      // outside the cache or the output: recorded, nothing written
    if (status && w == 0) atomicCAS(status, 0, RLB_ERR_BAD_ARG);
    return;
  }
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (slot >= 0) {
    const bool value = h >= Hkv;
    const long long blk = slot / block_size;
    const int off = static_cast<int>(slot - blk * block_size);
    const uint8_t* page = cache + (blk * Hkv + (value ? h - Hkv : h)) * Page::bytes(block_size);
    uint32_t c_lo, c_hi;
    if (value) {
      const uint8_t* v = page + Page::values_at(block_size);
      c_lo = *reinterpret_cast<const uint16_t*>(v + Page::value_unit(off, 2 * t, g)) | *reinterpret_cast<const uint16_t*>(v + Page::value_unit(off, 2 * t + 1, g)) << 16;
      c_hi = *reinterpret_cast<const uint16_t*>(v + Page::value_unit(off, 2 * t, g + UP)) | *reinterpret_cast<const uint16_t*>(v + Page::value_unit(off, 2 * t + 1, g + UP)) << 16;
    } else {
      c_lo = *reinterpret_cast<const uint32_t*>(page + Page::key_word(off, t, g));
      c_hi = *reinterpret_cast<const uint32_t*>(page + Page::key_word(off, t, g + UP));
    }
    const uint8_t* s = page + Page::scales_at(block_size);
    lo = values8(c_lo, *reinterpret_cast<const uint16_t*>(s + Page::scale(off, value, g)));
    hi = values8(c_hi, *reinterpret_cast<const uint16_t*>(s + Page::scale(off, value, g + UP)));
  }
  uint4* p = reinterpret_cast<uint4*>(out + to * out_stride + static_cast<long long>(h) * D + c * 8);
  p[0] = lo;
  p[D / 16] = hi;
}

template <int D>
int launch_write(void* qkv, const int* pos, const float* inv_freq, const long long* slots, void* cache, long long T, int Hq, int Hkv, int block_size, long long row_stride,
                 long long num_blocks, int* status, cudaStream_t stream) {
  const int heads = Hq + 2 * Hkv, threads = 128, rows = 1, per_block = threads * 16 / D;
  const dim3 grid(static_cast<unsigned>((T + rows - 1) / rows), static_cast<unsigned>((heads + per_block - 1) / per_block));
  rlb_launch_pdl(kv4_write_kernel<D>, grid, dim3(threads), rows * D / 2 * sizeof(float2), stream, static_cast<__nv_bfloat16*>(qkv), pos, inv_freq, slots, static_cast<uint8_t*>(cache), T, Hq,
                 Hkv, block_size, row_stride, num_blocks * block_size, status, rows, per_block);
  return static_cast<int>(cudaGetLastError());
}

template <int D>
int launch_read(const void* cache, const long long* slots, const long long* out_rows, void* out, long long n, long long out_stride, long long num_out, int Hkv, int block_size,
                long long num_blocks, int* status, cudaStream_t stream) {
  const long long items = n * 2 * Hkv * (D / 16);
  rlb_launch_pdl(kv4_read_kernel<D>, dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, stream, static_cast<const uint8_t*>(cache), slots, out_rows,
                 static_cast<__nv_bfloat16*>(out), n, out_stride, num_out, Hkv, block_size, num_blocks * block_size, status);
  return static_cast<int>(cudaGetLastError());
}
bool bad_shape(int D, int Hkv, int block_size) { return (D != 64 && D != 128 && D != 256) || Hkv < 1 || block_size < 16 || block_size % 16 || block_size > KV4_MAX_BLOCK; }
}  // namespace

// qkv [T, (Hq + 2 Hkv) D] bf16, 16-byte aligned rows; pos [T]; inv_freq [D / 2]; slots [T] (block * block_size + offset; negative: rotate only); cache: see kv4.cuh.
RLB_API int rlb_rope_kv4_cache_write(void* qkv, const int* pos, const float* inv_freq, const long long* slots, void* cache, long long T, int Hq, int Hkv, int D, int block_size,
                                     long long row_stride, long long num_blocks, int* status, void* stream) {
  if (bad_shape(D, Hkv, block_size) || Hq < 0 || row_stride % 8 || ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(cache)) & 15)) return -2;
  if (T <= 0) return 0;
  if (T > 0x7fffffffll) return -3;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = D == 64 ? launch_write<64> : D == 128 ? launch_write<128> : launch_write<256>;
  return launch(qkv, pos, inv_freq, slots, cache, T, Hq, Hkv, block_size, row_stride, num_blocks, status, s);
}

// out [num_out, >= 2 Hkv D] bf16, 16-byte aligned rows; slots [n]; out_rows [n] or null (row i goes to row i).
RLB_API int rlb_kv4_cache_read(const void* cache, const long long* slots, const long long* out_rows, void* out, long long n, long long out_stride, long long num_out, int Hkv, int D,
                               int block_size, long long num_blocks, int* status, void* stream) {
  if (bad_shape(D, Hkv, block_size) || out_stride % 8 || ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(cache)) & 15)) return -2;
  if (n <= 0) return 0;
  if (n * 2 * Hkv * (D / 16) / 256 >= 0x7fffffffll) return -3;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = D == 64 ? launch_read<64> : D == 128 ? launch_read<128> : launch_read<256>;
  return launch(cache, slots, out_rows, out, n, out_stride, num_out, Hkv, block_size, num_blocks, status, s);
}
