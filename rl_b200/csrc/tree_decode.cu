// Attention of the rows of drafted tokens' trees over the paged key/value cache: softmax(scale q K^T) V for every row over its sequence's context and the tree rows that its
// mask names. One CTA per row and query head, tiles of 128 keys, online softmax in 32 bits.
//
// This file is compiled without fast math.
#include "common.cuh"

#include <math.h>

namespace {
using namespace rlb;

struct TreeArgs {
  const __nv_bfloat16* q;
  long long ldq;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int blocks, block, pages;
  const int* table;
  long long table_ld;
  const int* ctx;
  const int* cu;
  int B, T, max_rows, Hq, Hkv;
  const int* masks;      // null: a row sees the rows up to itself
  long long masks_ld;
  const int* positions;      // with window > 0
  int window;
  float scale;
  __nv_bfloat16* out;
  long long ldo;
  int* status;
};

constexpr int TR_TILE = 128;
template <int D>
__global__ void __launch_bounds__(TR_TILE)
tree_rows_attention_kernel(const TreeArgs a) {
  __shared__ float q[D], score[TR_TILE], red[32];
  __shared__ long long place[TR_TILE];
  const int j = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = h / (a.Hq / a.Hkv);
  pdl_sync();
  const int lo = min(max(a.cu[b], 0), a.T), n = min(min(max(a.cu[b + 1], lo), a.T) - lo, a.max_rows);
  if (j >= n) return;
  const long long t = lo + j;
  for (int i = tid; i < D; i += TR_TILE) q[i] = __bfloat162float(a.q[t * a.ldq + h * D + i]) * a.scale;
  const long long room = static_cast<long long>(a.pages) * a.block;
  const int ctx = static_cast<int>(min(static_cast<long long>(max(a.ctx[b], 0)), room)), keys = static_cast<int>(min(static_cast<long long>(ctx) + n, room));
  const int pos = a.window > 0 ? max(a.positions[t], ctx) : 0;
  float m = -INFINITY, l = 0.f, o[D / TR_TILE > 0 ? D / TR_TILE : 1] = {};
  for (int t0 = a.window > 0 ? max(0, ctx - a.window + 1) : 0; t0 < keys; t0 += TR_TILE) {
    const int c = t0 + tid;
    bool sees = c < keys;
    if (sees && c >= ctx) {
      const int i = c - ctx;
      sees = a.masks ? a.masks[t * a.masks_ld + (i >> 5)] >> (i & 31) & 1 : i <= j;
      if (a.window > 0) sees = sees && pos - a.positions[lo + i] < a.window;
    } else if (sees && a.window > 0) {
      sees = pos - c < a.window;
    }
    __syncthreads();
    if (sees) {
      const int id = a.table[b * a.table_ld + c / a.block];
      if (id < 0 || id >= a.blocks) {
        if (a.status) atomicCAS(a.status, 0, RLB_ERR_BOUNDS);
        sees = false;
      } else {
        place[tid] = ((static_cast<long long>(id) * a.Hkv + g) * a.block + c % a.block) * D;
      }
    }
    if (!sees) place[tid] = -1;
    __syncthreads();
    for (int i = warp; i < TR_TILE; i += 4) {
      float s = 0.f;
      if (place[i] >= 0)
        for (int e = lane; e < D; e += 32) s = fmaf(q[e], __bfloat162float(a.k[place[i] + e]), s);
      s = warp_sum(s);
      if (lane == 0) score[i] = place[i] >= 0 ? s : -INFINITY;
    }
    __syncthreads();
    const float mine = score[tid], top = fmaxf(m, block_max(mine, red));
    const float p = top == -INFINITY ? 0.f : expf(mine - top), f = top == -INFINITY ? 1.f : expf(m - top);
    l = l * f + block_sum(p, red);
    m = top;
    __syncthreads();
    score[tid] = p;
    __syncthreads();
    if (tid < D) {
      float s = 0.f;
      for (int i = 0; i < TR_TILE; ++i)
        if (place[i] >= 0) s = fmaf(score[i], __bfloat162float(a.v[place[i] + tid]), s);
      o[0] = o[0] * f + s;
    }
  }
  if (tid < D) a.out[t * a.ldo + h * D + tid] = __float2bfloat16(l == 0.f ? 0.f : o[0] / l);
}
}  // namespace

RLB_API int rlb_tree_decode(const void* q, long long ldq, const void* k, const void* v, int blocks, int block, const int* table, long long table_ld, int pages,
                            const int* ctx, const int* cu, int B, int T, int max_rows, int Hq, int Hkv, int D, const int* masks, long long masks_ld,
                            const int* positions, int window, float scale, void* out, long long ldo, int* status, void* stream) {
  if (D != 64 && D != 128) return -2;
  if (Hkv < 1 || Hq % Hkv || Hq > 65535 || B > 65535) return -2;
  const TreeArgs a{static_cast<const __nv_bfloat16*>(q), ldq, static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v), blocks, block, pages, table,
                   table_ld, ctx, cu, B, T, max_rows, Hq, Hkv, masks, masks_ld, positions, window, scale, static_cast<__nv_bfloat16*>(out), ldo, status};
  return static_cast<int>(rlb_launch_pdl(D == 64 ? tree_rows_attention_kernel<64> : tree_rows_attention_kernel<128>, dim3(max_rows, Hq, B), dim3(TR_TILE), 0,
                                         static_cast<cudaStream_t>(stream), a));
}
