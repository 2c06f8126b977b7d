// What the kernels of the 4-bit key/value cache share: where a page keeps what.
//
// The cache is [num_blocks, Hkv, page bytes]: a page holds `block_size` tokens (a multiple of 16) of one key/value head of D dimensions (64, 128
// or 256), G = D / 32 groups of 32 consecutive dimensions each. A group is held as 32 codes of 4 bits and one bf16 scale:
//     a = max |x|,  s = bf16(a / 7.5)  (0 where a < 2^-100, NaN where a value of the group is not finite),
//     code = clamp(floor(x / s) + 8, 0, 15),  which stands for (code - 7.5) * s:
// 16 equally spaced levels, symmetric around zero, at most s / 2 from x. With a level on zero the outermost one on one side would be unused.
//
// Page: [keys' codes, block_size * D / 2 B][values' codes, the same][scales, block_size * D / 8 B]. Codes stand in 16-bit units of four consecutive
// dimensions (the first in the low bits) that are placed as the tensor-core instructions of the decode kernel want them, without a shuffle:
//   keys    token: [4 t][G groups][2] units; unit (t, g, h) holds dimensions 32 g + 8 t + 4 h .. + 3
//   values  two tokens: [8 r][G groups][2 tokens] units; unit (r, g, token) holds dimensions 32 g + 4 r .. + 3 of that token
//   scales  token: [keys, values][G] bf16
#pragma once

#include "common.cuh"

#include <atomic>

namespace rlb {

constexpr int KV4_GROUP = 32;
constexpr int KV4_MAX_BLOCK = 65536;      // places within a page are 32-bit offsets

// The current device (by which launchers keep what they have asked for) and its multiprocessors.
constexpr int KV4_DEVICES = 64;
inline cudaError_t kv4_device(int& dev, int& sms) {
  static std::atomic<int> known[KV4_DEVICES];
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= KV4_DEVICES) return cudaErrorInvalidDevice;
  sms = known[dev].load();
  if (sms) return cudaSuccess;
  const cudaError_t asked = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (asked == cudaSuccess) known[dev].store(sms);
  return asked;
}

template <int D>
struct Kv4Page {
  static constexpr int G = D / KV4_GROUP;
  __host__ __device__ static constexpr long long bytes(int block_size) { return static_cast<long long>(block_size) * D * 9 / 8; }
  __host__ __device__ static constexpr int values_at(int block_size) { return block_size * (D / 2); }
  __host__ __device__ static constexpr int scales_at(int block_size) { return block_size * D; }
  // 32-bit word of eight dimensions 32 g + 8 t .. + 7 of a key
  __host__ __device__ static constexpr int key_word(int token, int t, int g) { return token * (D / 2) + (t * G + g) * 4; }
  // 16-bit unit of four dimensions 32 g + 4 r .. + 3 of a value, within the values' part
  __host__ __device__ static constexpr int value_unit(int token, int r, int g) { return (token >> 1) * D + (r * G + g) * 4 + (token & 1) * 2; }
  __host__ __device__ static constexpr int scale(int token, int value, int g) { return (token * 2 + value) * (G * 2) + g * 2; }
};

}  // namespace rlb
