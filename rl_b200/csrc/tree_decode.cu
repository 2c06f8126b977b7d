// Attention of the rows of drafted tokens' trees over the paged key/value cache, on the 5th-generation tensor cores:
//   o[t, h] = sum_k w_k v_k / sum_k w_k,   w_k = exp(scale q[t, h] . k_k)
// over the keys that row t sees: its sequence's context, and of the tree's own rows (which stand behind it in the cache) those whose bits its mask has.
//
// The query heads of a key/value head and the rows of a tree are the M side of both products: row r of a block is head r % G of row r / G (G = Hq / Hkv), up to 128 / G rows of the
// tree to a block, which one TMA box [G heads x rows] brings. A unit is a block of one sequence and key/value head; its keys go by in tiles of 64:
//   warp 0      TMA producer: the unit's queries, then K tiles through a ring and V tiles through another. A tile is 64 / R boxes of R = gcd(page, 64) keys; a box whose page is not
//               there (behind the last key, or no page of the cache) starts behind the cache's last row, and arrives as zeros
//   warp 1      tcgen05.mma issuer: S = Q K^T (128 x 64 x D) into one of two TMEM buffers, one tile ahead of the softmax, then O += P V (128 x D x 64) with P read from TMEM
//   warps 2..5  softmax, a thread per row: maximum and sum in 32 bits; P is rounded to bf16 (half a step: up to 2^-8 of a weight, as the output's own rounding)
//               over the scores that were read; O is rescaled only when the maximum moved by more than 2^8.
// In tiles that some row does not see as a whole (the tree's, the window's edge, the last) a row has a word of 64 bits, and V is searched for values that are not finite: these would
// reach every row through weights of zero. They are set to zero there and added in the end to the rows that see them.
//
// The tiles of all units form one sequence, of which each CTA takes an equal share (two CTAs to an SM, all resident): contexts of any lengths fill the device. Units that
// are cut leave sums, maximum and 32-bit output of their parts in a workspace, and a second kernel joins them in their order. With few tiles to a unit a CTA takes a whole unit instead.
//
// Long contexts of few rows are bound by memory (31 chains of 5 on 32768 tokens, 32 / 8 heads of 128: 4.2 GB of keys and values, 637 us at the rate of a plain copy: 605 in a graph of short runs,
// 670 to 741 in calls one after another, board by board). With 64 rows and more the
// tensor cores and the softmax take turns: a product of 64 keys costs as much as one of 128, and a pair of tiles takes 2100 cycles, 1540 of them the products' (16 trees of 64 on 8001, 28 / 4 heads: 103 us,
// 0.17 GB; one tree of 33 on 131072, 40 / 8 heads: 152 us, 0.54 GB). Short contexts pay for a unit's start and end (64 trees of 17 rows to 1280 tokens: 52 us where memory takes 35).
//
// This file is compiled without fast math.
#include "common.cuh"

#include <math.h>

namespace {
using namespace rlb;

constexpr int M_ROWS = 128, TILE = 64;
constexpr int THREADS = 192;
constexpr int TMEM_COLS = 256;      // scores of even and odd tiles at columns 0 and 64, P and the output where Shape says
constexpr int BAD_RING = 8;         // the producer is at most four tiles ahead of the softmax
constexpr float RESCALE = 8.f;      // log2
constexpr float LOG2E_F = 1.4426950408889634f;

struct Cut;
struct TreeArgs {
  int blocks, block, block_shift, pages, box;      // block_shift: of pages of a power of two, else -1; box: keys of a TMA box
  const int* table;
  long long table_ld;
  const int* ctx;
  const int* cu;
  int B, T, max_rows, Hq, Hkv, G;
  int block_rows, block_inv, group_inv, q_rows;      // tree rows of a block, 65536 / that and one, the same of G, rows of a TMA box of queries
  const int* masks;            // null: a row sees the rows up to itself
  long long masks_ld;
  const int* positions;        // with window > 0
  int window;
  float scale_log2;
  __nv_bfloat16* out;
  long long ldo;
  int vec;                     // rows of `out` start on 32 bytes
  const __nv_bfloat16* v;
  float* part_o;               // [2 CTAs][part_rows][D]: first and last part of a CTA; null: a CTA has a whole unit
  float2* part_ml;             // [2 CTAs][part_rows] maximum (log2) and sum
  Cut* cuts;                   // [CTAs]
  int part_rows, least;        // least: tiles of a share at least
  int group;                   // CTAs beside one another that have the same tiles, each a block of its own
  int sorted;                  // whole units: in order of their sequences' lengths (at most THREADS of them)
  int* status;
};

template <int D>
struct Shape {
  static constexpr int ATOMS = D / 64;
  static constexpr int K_STAGES = D == 128 ? 3 : 5, V_STAGES = D == 128 ? 2 : 4;
  static constexpr int Q_ATOM = M_ROWS * 128, KV_ATOM = TILE * 128;
  static constexpr int Q_BYTES = ATOMS * Q_ATOM, KV_BYTES = ATOMS * KV_ATOM;
  // P over the scores that were read, where the output leaves no room for places of its own: the scores after next then wait for the product
  static constexpr bool OWN_P = D == 64;
  static constexpr int P_COL = OWN_P ? 128 : 0, P_STEP = OWN_P ? 32 : 64, O_COL = OWN_P ? 192 : 128;
  static constexpr int SMEM = Q_BYTES + (K_STAGES + V_STAGES) * KV_BYTES + 512;
};

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// 32 bytes at once: whole sectors, although a warp's lanes write rows of their own.
__device__ __forceinline__ void store32(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f, uint32_t g, uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e), "r"(f), "r"(g), "r"(h) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {      // relative error 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Most waits have nothing to wait for: the rest of them is out of line (84 KB of instructions with all of it in place, for which a unit's few thousand ones that run once
// came from the second level cache: some 6000 cycles).
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  return mbar_wait(bar, parity, abort_flag, status, code);
}
__device__ __forceinline__ bool one_wait(const uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  return mbar_try_wait(smem_u32(bar), parity) || wait_long(smem_u32(bar), parity, abort_flag, status, code);
}
// A whole warp waits: all of its lanes go on, or none.
__device__ __forceinline__ bool warp_wait(const uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  return __all_sync(0xffffffffu, one_wait(bar, parity, abort_flag, status, code));
}

// A sequence's rows and keys, and its units' tiles.
struct Seq {
  int lo, n, ctx, keys, first, tiles, blocks;      // first: the first tile that is in the window
};
__device__ __noinline__ Seq sequence(const TreeArgs& a, int b) {
  Seq s;
  s.lo = min(max(a.cu[b], 0), a.T);
  s.n = min(min(max(a.cu[b + 1], s.lo), a.T) - s.lo, a.max_rows);
  const int room = a.pages * a.block;      // at most 2^31 - 2^16
  s.ctx = min(max(a.ctx[b], 0), room);
  s.keys = s.n > 0 ? s.ctx + min(s.n, room - s.ctx) : 0;
  s.first = a.window > 0 ? max(0, s.ctx - a.window + 1) / TILE : 0;
  s.blocks = ((s.n + a.block_rows - 1) * a.block_inv) >> 16;      // (exact: less than 384 over at most 128)
  s.tiles = max((s.keys + TILE - 1) / TILE - s.first, s.n > 0 ? 1 : 0);      // (rows without any key have a tile too, which they do not see)
  return s;
}
__device__ __forceinline__ int tiles_of(const TreeArgs& a, const Seq& s) { return s.tiles * (a.group > 1 ? min(s.blocks, 1) : s.blocks) * a.Hkv; }      // (shared tiles are less than 2^31 in all)

// Sums over the block's threads: of those before this one, and of all. `red`: a word for each warp.
__device__ __forceinline__ int block_scan(int v, int* red, int& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += u;
  }
  __syncthreads();
  if (lane == 31) red[warp] = run;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const int x = red[w];
    if (w < warp) before += x;
    all += x;
  }
  return before + run - v;
}
// What a CTA's first part is the rest of: how many of the unit's tiles came before it (0: nothing), and of how many.
struct Cut {
  int share;            // tiles of a CTA
  int row, rows, head;  // of the output, of the unit; first head
  int before, tiles, none[2];
};

struct Segment {      // what a CTA does of one unit
  Seq s;
  int b, kv_head, j0, rows;      // first row of the tree, rows of the block's M side
  int t0, t1;                    // tiles of the unit
  bool whole;
};
struct Cursor {
  int left;                // tiles that this CTA still has
  int b, kv_head, m, t;    // sequence, unit and tile that come next
  Seq s;
  __device__ __forceinline__ bool next(const TreeArgs& a, Segment& g) {
    if (left <= 0) return false;
    if (t == s.tiles) {
      t = 0;
      if (a.group > 1 || ++m == s.blocks) {
        if (a.group <= 1) m = 0;
        ++kv_head;
      }
    }
    while (s.blocks == 0 || kv_head == a.Hkv || m >= s.blocks) {
      if (kv_head < a.Hkv && s.blocks > 0) {      // a sequence without a block of this number
        left -= (a.Hkv - kv_head) * s.tiles - t;
        if (left <= 0) return false;
      }
      kv_head = t = 0;
      if (++b >= a.B) return false;
      s = sequence(a, b);
    }
    g.s = s;
    g.b = b;
    g.kv_head = kv_head;
    g.j0 = m * a.block_rows;
    g.rows = min(a.block_rows, s.n - g.j0) * a.G;
    g.t0 = t;
    g.t1 = min(s.tiles - t, left) + t;
    g.whole = g.t0 == 0 && g.t1 == s.tiles;
    left -= g.t1 - g.t0;
    t = g.t1;
    return true;
  }
};

// Which of the tile's keys a row sees.
struct RowView {
  const int* mask;      // null: a chain
  int words, j, pos;
  uint32_t w0, w1;      // its first two words
};
__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }
__device__ __noinline__ uint64_t seen_keys(const TreeArgs& a, int ctx, int keys, int lo, int n, const RowView r, int k0) {
  uint64_t v = low_bits(keys - k0);
  const int base = k0 - ctx;      // row of the tree at bit 0
  if (base > -TILE) {
    uint64_t tree;
    const int from = max(base, 0);
    if (r.mask && from == 0) {
      tree = r.w0 | static_cast<uint64_t>(r.w1) << 32;
    } else if (r.mask) {
      const int w = from >> 5, sh = from & 31;
      const uint64_t w0 = w < r.words ? static_cast<uint32_t>(r.mask[w]) : 0u, w1 = w + 1 < r.words ? static_cast<uint32_t>(r.mask[w + 1]) : 0u,
                     w2 = w + 2 < r.words ? static_cast<uint32_t>(r.mask[w + 2]) : 0u;
      tree = (w0 | w1 << 32) >> sh;
      if (sh) tree |= w2 << (64 - sh);
    } else {
      tree = low_bits(r.j - from + 1);
    }
    v &= base < 0 ? low_bits(-base) | tree << -base : tree;
  }
  if (a.window > 0) {
    const int behind = min(r.pos - a.window + 1, ctx) - k0;      // context keys before it are not in the window
    v &= ~low_bits(behind);
    if (base > -TILE) {
      for (int i = max(0, -base); i < TILE && base + i < n; ++i)
        if (r.pos - a.positions[lo + base + i] >= a.window) v &= ~(1ull << i);
    }
  }
  return v;
}

// 16 keys of the tile each that have no page of the cache.
__device__ __forceinline__ uint64_t without_pages(uint64_t v, int bad) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (bad >> i & 1) v &= ~(0xffffull << (16 * i));
  return v;
}

__device__ __forceinline__ float max3(float a, float b, float c) {      // of those that are numbers
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two at a time.
__device__ __forceinline__ uint64_t pair(float a, float b) { return static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float low_of(uint64_t a) { return __uint_as_float(static_cast<uint32_t>(a)); }
__device__ __forceinline__ float high_of(uint64_t a) { return __uint_as_float(static_cast<uint32_t>(a >> 32)); }
__device__ __forceinline__ bool not_finite(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

// Adds values that are not finite, of tiles that some row does not see as a whole, to the row that sees them: to its output, or to its part.
template <int D>
__device__ __noinline__ void add_special(const TreeArgs& a, const Segment g, const RowView view, int edge, __nv_bfloat16* dst, float* part) {
  for (int t = g.t0; t < g.t1; ++t) {
    const int k0 = (g.s.first + t) * TILE;
    int lost = 0;
    for (int i = 0; i < TILE && k0 + i < g.s.keys; i += 16) {
      const int id = a.table[g.b * a.table_ld + (k0 + i) / a.block];
      if (id < 0 || id >= a.blocks) lost |= 1 << (i >> 4);
    }
    if (k0 + TILE <= g.s.ctx && k0 >= edge && !lost) continue;
    const uint64_t seen = without_pages(seen_keys(a, g.s.ctx, g.s.keys, g.s.lo, g.s.n, view, k0), lost);
    for (int i = 0; i < TILE; ++i) {
      if (!(seen >> i & 1)) continue;
      const int id = a.table[g.b * a.table_ld + (k0 + i) / a.block];
      const __nv_bfloat16* v = a.v + ((static_cast<long long>(id) * a.Hkv + g.kv_head) * a.block + (k0 + i) % a.block) * D;
      for (int e = 0; e < D; ++e) {
        const float x = __bfloat162float(v[e]);
        if (fabsf(x) < INFINITY) continue;
        if (part) part[e] += x;
        else dst[e] = __float2bfloat16(__bfloat162float(dst[e]) + x);
      }
    }
  }
}

// The first row of a sequence's box in the cache, -1 without a page, -2 behind the keys.
__device__ __noinline__ int look(const TreeArgs& a, const int* table, int kv_head, int keys, int box) {
  const long long key = static_cast<long long>(box) * a.box;
  if (key >= keys) return -2;
  const int k = static_cast<int>(key), page = a.block_shift >= 0 ? k >> a.block_shift : k / a.block, id = table[page];
  if (id < 0 || id >= a.blocks) {
    if (a.status) atomicCAS(a.status, 0, RLB_ERR_BOUNDS);
    return -1;
  }
  return (id * a.Hkv + kv_head) * a.block + (k - page * a.block);
}

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
tree_decode_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ TreeArgs a) {
  using S = Shape<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* q_s = smem;
  uint8_t* k_s = q_s + S::Q_BYTES;
  uint8_t* v_s = k_s + S::K_STAGES * S::KV_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + S::V_STAGES * S::KV_BYTES);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* o_empty = bars + 2;
  uint64_t* s_full = bars + 3;        // [2]
  uint64_t* p_full = bars + 5;        // [2]
  uint64_t* k_full = bars + 7;        // [K_STAGES]
  uint64_t* k_empty = k_full + S::K_STAGES;
  uint64_t* v_full = k_empty + S::K_STAGES;
  uint64_t* v_empty = v_full + S::V_STAGES;      // also: the product with this V tile is in O
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_empty + S::V_STAGES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* special = abort_flag + 1;      // [2] last even and odd unit with values that are not finite in a tile that some row does not see as a whole
  volatile int* bad = special + 2;             // [BAD_RING]
  int* red = reinterpret_cast<int*>(smem + S::SMEM - 128);      // [THREADS / 32]
  int* start = red + THREADS / 32;                              // [2]

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // (one of the warp's, as the compiler sees then)
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
    mbar_init(smem_u32(q_full), 1);
    mbar_init(smem_u32(q_empty), 1);
    mbar_init(smem_u32(o_empty), 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&p_full[i]), 4);
    }
    for (int i = 0; i < S::K_STAGES; ++i) {
      mbar_init(smem_u32(&k_full[i]), 1);
      mbar_init(smem_u32(&k_empty[i]), 1);
    }
    for (int i = 0; i < S::V_STAGES; ++i) {
      mbar_init(smem_u32(&v_full[i]), 1);
      mbar_init(smem_u32(&v_empty[i]), 1);
    }
    *abort_flag = 0;
    special[0] = special[1] = -1;
    mbar_fence_init();
    fence_proxy_async();
  }
  __syncthreads();      // (no warp waits for a barrier before it is one, whichever way it goes below)
  pdl_sync();

  // ---------------------------------------------------------------- this CTA's tiles
  Cursor cur;
  if (a.part_o) {
    int total = 0, before = 0, mine = 0, all;      // of all sequences, of those before this thread's, of its own
    for (int b0 = 0; b0 < a.B; b0 += THREADS) {
      const int b = b0 + threadIdx.x;
      mine = b < a.B ? tiles_of(a, sequence(a, b)) : 0;
      before = total + block_scan(mine, red, all);
      total += all;
    }
    const unsigned groups = gridDim.x / a.group, mine_of = blockIdx.x / a.group;
    const int share = max(a.least, static_cast<int>((static_cast<unsigned>(total) + groups - 1) / groups));
    const long long from = static_cast<long long>(share) * mine_of;
    if (from >= total) {
      if (threadIdx.x == 0) a.cuts[blockIdx.x].before = 0;
      return;
    }
    const int begin = static_cast<int>(from);
    if (a.B > THREADS) {      // the sequence that it lies in once more
      int sofar = 0;
      for (int b0 = 0; b0 < a.B && sofar <= begin; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        mine = b < a.B ? tiles_of(a, sequence(a, b)) : 0;
        before = sofar + block_scan(mine, red, all);
        sofar += all;
        if (begin >= before && begin < before + mine) start[0] = b;
        if (begin >= before && begin < before + mine) start[1] = begin - before;
      }
    } else if (begin >= before && begin < before + mine) {
      start[0] = threadIdx.x;
      start[1] = begin - before;
    }
    __syncthreads();
    cur.b = start[0];
    cur.s = sequence(a, cur.b);
    const int unit = start[1] / cur.s.tiles;
    cur.t = start[1] - unit * cur.s.tiles;
    if (a.group > 1) {
      cur.kv_head = unit;
      cur.m = blockIdx.x - mine_of * a.group;
    } else {
      cur.kv_head = unit / cur.s.blocks;
      cur.m = unit - cur.kv_head * cur.s.blocks;
    }
    cur.left = min(share, total - begin);
    if (threadIdx.x == 0) {
      const int j0 = cur.m * a.block_rows;
      a.cuts[blockIdx.x] = Cut{share, cur.s.lo + j0, min(a.block_rows, cur.s.n - j0) * a.G, cur.kv_head * a.G, cur.m < cur.s.blocks ? cur.t : 0, cur.s.tiles, {0, 0}};
    }
  } else {
    cur.b = blockIdx.z;
    if (a.sorted) {      // the longest sequences' units first: the last ones to run are short
      int* keys = reinterpret_cast<int*>(smem);      // (the loads' place)
      const int b = threadIdx.x;
      int mine = 0;
      if (b < a.B) {
        const Seq s = sequence(a, b);
        keys[b] = mine = s.n > 0 ? s.tiles : 0;
      }
      __syncthreads();
      int before = 0;
      for (int i = 0; i < a.B; ++i) before += keys[i] > mine || (keys[i] == mine && i < b);
      if (b < a.B && before == static_cast<int>(blockIdx.z)) start[0] = b;
      __syncthreads();
      cur.b = start[0];
      fence_proxy_async();
    }
    if (threadIdx.x == 0 && a.window == 0) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.table + cur.b * a.table_ld));
    cur.s = sequence(a, cur.b);
    if (static_cast<int>(blockIdx.x) >= cur.s.blocks) return;
    cur.kv_head = blockIdx.y;
    cur.m = blockIdx.x;
    cur.t = 0;
    cur.left = cur.s.tiles;
  }
  if (smem_u32(smem) & 1023u) {      // the swizzled tiles need a base of 1024 bytes; report instead of misreading
    if (threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, RLB_ERR_BAD_ARG);
    return;
  }
  uint32_t tmem_base = 0, tmem_o = 0;
  if (warp != 0) {      // (the loads need not wait for this)
    if (warp == 1) {
      tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
      tmem_relinquish();
    }
    tc_fence_before();
    asm volatile("bar.sync 1, 160;" ::: "memory");
    tc_fence_after();
    tmem_base = *tmem_slot;
    tmem_o = tmem_base + S::O_COL;
  }

  Segment g;
  if (warp == 0) {
    // ------------------------------------------------------------ loads
    const int boxes = TILE / a.box, end_row = a.blocks * a.Hkv * a.block;      // (behind the last row: zeros)
    const uint32_t q_bytes = static_cast<uint32_t>(a.q_rows) * a.G * 128 * S::ATOMS;
    bool ok = true;
    int it = 0;
    for (int unit = 0; ok && cur.next(a, g); ++unit) {
      const int* table = a.table + g.b * a.table_ld;
      // lane i has the first row of box i of the next 32, and one more of those behind them
      int at = (g.s.first + g.t0) * boxes, rows = look(a, table, g.kv_head, g.s.keys, at + lane), ahead = -2, used = 0;
      if (unit > 0) ok = warp_wait(q_empty, (unit - 1) & 1, abort_flag, a.status, RLB_ERR_WAIT_EMPTY);
      if (!ok) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(smem_u32(q_full), q_bytes);
#pragma unroll
        for (int c = 0; c < S::ATOMS; ++c) tma_load_3d(smem_u32(q_s + c * S::Q_ATOM), &tmap_q, smem_u32(q_full), c * 64, g.kv_head * a.G, g.s.lo + g.j0);
      }
      __syncwarp();
      for (int t = g.t0; t < g.t1 && ok; ++t, ++it) {
        const int ks = it % S::K_STAGES, vs = it % S::V_STAGES;
        if (used == 32) {
          used = 0;
          at += 32;
          rows = ahead;
        }
        int row[4], lost = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          row[i] = i < boxes ? __shfl_sync(0xffffffffu, rows, used + i) : 0;
          if (i < boxes && row[i] == -1) lost |= ((1 << (a.box >> 4)) - 1) << (i * (a.box >> 4));
          if (row[i] < 0) row[i] = end_row;
        }
        used += boxes;
        const bool more = used == boxes;      // (the next ones while these are loaded)
        ok = warp_wait(&k_empty[ks], ((it / S::K_STAGES) & 1) ^ 1, abort_flag, a.status, RLB_ERR_WAIT_EMPTY);
        if (!ok) break;
        if (elect_one()) {
          bad[it % BAD_RING] = lost;
          mbar_arrive_expect_tx(smem_u32(&k_full[ks]), S::KV_BYTES);
#pragma unroll
          for (int c = 0; c < S::ATOMS; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i < boxes) tma_load_2d(smem_u32(k_s + ks * S::KV_BYTES + c * S::KV_ATOM + i * a.box * 128), &tmap_k, smem_u32(&k_full[ks]), c * 64, row[i]);
        }
        __syncwarp();
        if (more) ahead = look(a, table, g.kv_head, g.s.keys, at + 32 + lane);
        ok = warp_wait(&v_empty[vs], ((it / S::V_STAGES) & 1) ^ 1, abort_flag, a.status, RLB_ERR_WAIT_EMPTY);
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(smem_u32(&v_full[vs]), S::KV_BYTES);
#pragma unroll
          for (int c = 0; c < S::ATOMS; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i < boxes) tma_load_2d(smem_u32(v_s + vs * S::KV_BYTES + c * S::KV_ATOM + i * a.box * 128), &tmap_v, smem_u32(&v_full[vs]), c * 64, row[i]);
        }
        __syncwarp();
      }
    }
    if (!ok) {      // loads in flight land within microseconds: they must not outlive the CTA
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000ull) {}
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_bf16(M_ROWS, TILE, false, false), idesc_o = make_idesc_bf16(M_ROWS, D, false, true);
      auto scores = [&](int it, bool last_of_unit) -> bool {      // its buffer held P of tile it - 2, whose product has to be complete
        const int ks = it % S::K_STAGES;
        if (!S::OWN_P && it > 1 && !one_wait(&v_empty[(it - 2) % S::V_STAGES], ((it - 2) / S::V_STAGES) & 1, abort_flag, a.status, RLB_ERR_WAIT_TMEM_EMPTY))
          return false;
        if (!one_wait(&k_full[ks], (it / S::K_STAGES) & 1, abort_flag, a.status, RLB_ERR_WAIT_FULL)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t qa = smem_u32(q_s) + (kk / 4) * S::Q_ATOM + (kk % 4) * 32, ka = smem_u32(k_s + ks * S::KV_BYTES) + (kk / 4) * S::KV_ATOM + (kk % 4) * 32;
          umma_f16(tmem_base + (it & 1) * 64, make_smem_desc_sw128(qa, 16, 1024), make_smem_desc_sw128(ka, 16, 1024), idesc_s, kk != 0 ? 1u : 0u);
        }
        umma_commit(smem_u32(&s_full[it & 1]));
        umma_commit(smem_u32(&k_empty[ks]));
        if (last_of_unit) umma_commit(smem_u32(q_empty));
        return true;
      };
      bool ok = true;
      int it = 0;
      for (int unit = 0; ok && cur.next(a, g); ++unit) {
        const int n = g.t1 - g.t0;
        ok = one_wait(q_full, unit & 1, abort_flag, a.status, RLB_ERR_WAIT_FULL);
        for (int t = -1; t < n && ok; ++t) {      // the scores of tile t + 1, the output of tile t
          if (t + 1 < n && !scores(it + t + 1, t + 2 == n)) ok = false;
          if (t < 0) continue;
          const int i = it + t, vs = i % S::V_STAGES;
          if (ok && t == 0 && unit > 0) ok = one_wait(o_empty, (unit - 1) & 1, abort_flag, a.status, RLB_ERR_WAIT_TMEM_EMPTY);
          ok = ok && one_wait(&p_full[i & 1], (i >> 1) & 1, abort_flag, a.status, RLB_ERR_WAIT_FLAG) &&
               one_wait(&v_full[vs], (i / S::V_STAGES) & 1, abort_flag, a.status, RLB_ERR_WAIT_FULL);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < TILE / 16; ++kk)      // 16 keys each, 8 columns of P
            umma_f16_ts(tmem_o, tmem_base + S::P_COL + (i & 1) * S::P_STEP + kk * 8, make_smem_desc_sw128(smem_u32(v_s + vs * S::KV_BYTES) + kk * (16 * 128), S::KV_ATOM, 1024), idesc_o,
                        (t | kk) != 0 ? 1u : 0u);
          umma_commit(smem_u32(&v_empty[vs]));
        }
        it += n;
      }
    }
  } else {
    // ------------------------------------------------------------ softmax: a thread per row
    const int quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int own_j = (r * a.group_inv) >> 16, own_h = r - own_j * a.G;
    const bool neg = a.scale_log2 < 0.f;
    const float hidden = neg ? INFINITY : -INFINITY, size = fabsf(a.scale_log2);
    bool ok = true;
    int it = 0;
    for (int unit = 0; ok && cur.next(a, g); ++unit) {
      const bool active = quarter * 32 < g.rows;      // of the warp
      const int j = min(g.j0 + own_j, g.s.n - 1);   // (rows behind the block's compute as its last one)
      RowView view{a.masks ? a.masks + (g.s.lo + j) * a.masks_ld : nullptr, (a.max_rows + 31) >> 5, j, a.window > 0 ? max(a.positions[g.s.lo + j], g.s.ctx) : 0, 0u, 0u};
      if (a.masks) {      // (on their way while the first tiles go by)
        view.w0 = static_cast<uint32_t>(view.mask[0]);
        view.w1 = view.words > 1 ? static_cast<uint32_t>(view.mask[1]) : 0u;
      }
      int edge = 0;      // keys before it are out of some row's window
      if (a.window > 0) {
        int far = g.s.ctx;
        for (int i = lane; i < a.block_rows && g.j0 + i < g.s.n; i += 32) far = max(far, a.positions[g.s.lo + g.j0 + i]);
        edge = __reduce_max_sync(0xffffffffu, far) - a.window + 1;
      }
      float m_ref = -INFINITY, l = 0.f;
      for (int t = g.t0; t < g.t1; ++t, ++it) {
        const uint32_t tmem_s = tmem_base + (it & 1) * 64 + lane_addr;
        const int k0 = (g.s.first + t) * TILE;
        if (!warp_wait(&s_full[it & 1], (it >> 1) & 1, abort_flag, a.status, RLB_ERR_WAIT_TMEM_FULL)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int lost = bad[it % BAD_RING];
        const bool cut = k0 + TILE > g.s.ctx || k0 < edge || lost;      // some row does not see some key
        if (active) {
          uint32_t s0[32], s1[32];
          tmem_ld_32x32b_x32(tmem_s, s0);
          tmem_ld_32x32b_x32(tmem_s + 32, s1);
          tmem_ld_wait();
          if (cut) {
            const uint64_t seen = without_pages(seen_keys(a, g.s.ctx, g.s.keys, g.s.lo, g.s.n, view, k0), lost);
            const uint32_t lo = static_cast<uint32_t>(seen), hi = static_cast<uint32_t>(seen >> 32);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (!(lo >> i & 1)) s0[i] = __float_as_uint(hidden);
              if (!(hi >> i & 1)) s1[i] = __float_as_uint(hidden);
            }
          }
          if (neg) {      // scores are compared before scaling
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              s0[i] ^= 0x80000000u;
              s1[i] ^= 0x80000000u;
            }
          }
          float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            best[0] = max3(best[0], __uint_as_float(s0[i]), __uint_as_float(s0[i + 1]));
            best[1] = max3(best[1], __uint_as_float(s0[i + 2]), __uint_as_float(s0[i + 3]));
            best[2] = max3(best[2], __uint_as_float(s1[i]), __uint_as_float(s1[i + 1]));
            best[3] = max3(best[3], __uint_as_float(s1[i + 2]), __uint_as_float(s1[i + 3]));
          }
          best[0] = max3(best[0], best[1], fmaxf(best[2], best[3]));
          const float mx = best[0] * size;
          float factor = 1.f;
          bool need = false;
          if (mx > m_ref + RESCALE || m_ref == -INFINITY) {
            const float m_new = fmaxf(mx, m_ref);
            if (m_new != -INFINITY) {
              factor = m_ref == -INFINITY ? 0.f : exp2_fast(m_ref - m_new);
              need = m_ref != -INFINITY;      // (nothing in O yet otherwise)
              m_ref = m_new;
            }
          }
          const float mr = m_ref == -INFINITY ? 0.f : -m_ref;
          const uint64_t size2 = pair(size, size), mr2 = pair(mr, mr);
          uint64_t sum[2] = {0ull, 0ull};
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t x = fma_pair(pair(__uint_as_float(s0[2 * i]), __uint_as_float(s0[2 * i + 1])), size2, mr2);
            const uint64_t y = fma_pair(pair(__uint_as_float(s1[2 * i]), __uint_as_float(s1[2 * i + 1])), size2, mr2);
            const float e0 = exp2_fast(low_of(x)), e1 = exp2_fast(high_of(x)), f0 = exp2_fast(low_of(y)), f1 = exp2_fast(high_of(y));
            pk[i] = pack_bf16x2(e0, e1);
            pk[16 + i] = pack_bf16x2(f0, f1);
            // (of the rounded weights: what a row's heaviest key lost by its rounding, the sum has lost too)
            sum[0] = add_pair(sum[0], pair(__uint_as_float(pk[i] << 16), __uint_as_float(pk[i] & 0xffff0000u)));
            sum[1] = add_pair(sum[1], pair(__uint_as_float(pk[16 + i] << 16), __uint_as_float(pk[16 + i] & 0xffff0000u)));
          }
          sum[0] = add_pair(sum[0], sum[1]);
          l = l * factor + (low_of(sum[0]) + high_of(sum[0]));
          // (the product with what stood there has been completed: these scores were issued after it)
          tmem_st_32x32b_x32(tmem_base + S::P_COL + (it & 1) * S::P_STEP + lane_addr, pk);
          if (__any_sync(0xffffffffu, need)) {
            // O may be touched only after the previous product has completed (the next one waits for p_full)
            if (!warp_wait(&v_empty[(it - 1) % S::V_STAGES], ((it - 1) / S::V_STAGES) & 1, abort_flag, a.status, RLB_ERR_WAIT_TMEM_EMPTY)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(tmem_o + lane_addr + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
              tmem_st_32x32b_x32(tmem_o + lane_addr + c * 32, o);
            }
          }
          tmem_st_wait();
          tc_fence_before();
        }
        if (cut) {
          const int vs = it % S::V_STAGES;
          if (!warp_wait(&v_full[vs], (it / S::V_STAGES) & 1, abort_flag, a.status, RLB_ERR_WAIT_FULL)) {
            ok = false;
            break;
          }
          uint4* v = reinterpret_cast<uint4*>(v_s + vs * S::KV_BYTES);
          bool found = false;
#pragma unroll 2
          for (int i = 0; i < S::KV_BYTES / 16 / 128; ++i) {
            uint4 x = v[i * 128 + r];
            if (not_finite(x.x) || not_finite(x.y) || not_finite(x.z) || not_finite(x.w)) {
              uint32_t* w = &x.x;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
                if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu;
              }
              v[i * 128 + r] = x;
              found = true;
            }
          }
          if (found) {
            special[unit & 1] = unit;
            fence_proxy_async();
          }
          __syncwarp();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[it & 1]));
      }
      if (!ok || !warp_wait(&v_empty[(it - 1) % S::V_STAGES], ((it - 1) / S::V_STAGES) & 1, abort_flag, a.status, RLB_ERR_WAIT_TMEM_EMPTY)) {
        ok = false;
        break;
      }
      if (active) {
        tc_fence_after();
        const bool there = r < g.rows;
        const long long slot = (2 * static_cast<long long>(blockIdx.x) + (g.t0 == 0)) * a.part_rows + r;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (there && !g.whole) a.part_ml[slot] = make_float2(m_ref, l);
        __nv_bfloat16* dst = a.out + (g.s.lo + j) * a.ldo + (g.kv_head * a.G + own_h) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld_32x32b_x32(tmem_o + lane_addr + c * 32, o);
          tmem_ld_wait();
          if (!there) continue;
          if (!g.whole) {
            float* to = a.part_o + slot * D + c * 32;
#pragma unroll
            for (int q = 0; q < 32; q += 8) store32(to + q, o[q], o[q + 1], o[q + 2], o[q + 3], o[q + 4], o[q + 5], o[q + 6], o[q + 7]);
            continue;
          }
          uint32_t w[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) w[q] = pack_bf16x2(__uint_as_float(o[2 * q]) * inv, __uint_as_float(o[2 * q + 1]) * inv);
          if (a.vec) {
#pragma unroll
            for (int q = 0; q < 16; q += 8) store32(dst + c * 32 + q * 2, w[q], w[q + 1], w[q + 2], w[q + 3], w[q + 4], w[q + 5], w[q + 6], w[q + 7]);
          } else {
#pragma unroll
            for (int q = 0; q < 16; ++q) {
              const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&w[q]);
              dst[c * 32 + 2 * q] = h.x;
              dst[c * 32 + 2 * q + 1] = h.y;
            }
          }
        }
        if (there && special[unit & 1] == unit) add_special<D>(a, g, view, edge, g.whole ? dst : nullptr, g.whole ? nullptr : a.part_o + slot * D);
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(o_empty));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Joins the parts of a unit that several CTAs had: a CTA for 8 of its rows, for each CTA whose first part is a unit's second.
constexpr int JOIN_ROWS = 8;
template <int D>
__global__ void __launch_bounds__(JOIN_ROWS * D / 8)
tree_join_kernel(const TreeArgs a) {
  pdl_sync();
  const int c = blockIdx.y, r = blockIdx.x * JOIN_ROWS + threadIdx.x / (D / 8), d = (threadIdx.x % (D / 8)) * 8;
  const Cut cut = a.cuts[c];
  if (cut.before == 0 || cut.before > cut.share || r >= cut.rows) return;
  const int last = c + (cut.tiles - cut.before - 1) / cut.share * a.group;
  float o[8] = {}, l = 0.f, top = -INFINITY;
#pragma unroll 2
  for (int k = c - a.group; k <= last; k += a.group) {      // the first one is its CTA's last part, the others their CTA's first
    const long long i = (2 * static_cast<long long>(k) + (k < c)) * a.part_rows + r;
    const float2 ml = a.part_ml[i];
    const float4 x = *reinterpret_cast<const float4*>(a.part_o + i * D + d), y = *reinterpret_cast<const float4*>(a.part_o + i * D + d + 4);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;      // nothing seen
    const float m = fmaxf(top, ml.x);
    const float f = top == -INFINITY ? 0.f : exp2f(top - m), w = ml.x == -INFINITY ? 1.f : exp2f(ml.x - m);      // (a sum beside no maximum is not a number)
    top = m;
    l = (f == 0.f ? 0.f : l * f) + (w == 0.f ? 0.f : ml.y * w);
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int q = 0; q < 8; ++q) o[q] = (f == 0.f ? 0.f : o[q] * f) + (w == 0.f ? 0.f : v[q] * w);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* dst = a.out + static_cast<long long>(cut.row + r / a.G) * a.ldo + (cut.head + r % a.G) * D + d;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(o[2 * i] * inv, o[2 * i + 1] * inv);
  if (a.vec) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
      dst[2 * i] = h.x;
      dst[2 * i + 1] = h.y;
    }
  }
}

int make_tmap_q(CUtensorMap* map, const void* q, uint64_t D, uint64_t heads, uint64_t rows, uint64_t ld_bytes, uint32_t box_heads, uint32_t box_rows) {
  RlbEncodeTiledFn encode = rlb_get_encode_tiled();
  if (!encode) return 1;
  const cuuint64_t dims[3] = {D, heads, rows}, strides[2] = {D * 2, ld_bytes};
  const cuuint32_t box[3] = {64, box_heads, box_rows}, unit[3] = {1, 1, 1};
  return static_cast<int>(encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
}

template <int D>
int launch(const void* q, long long ldq, const void* k, const void* v, TreeArgs a, int ctas, cudaStream_t stream) {
  CUtensorMap tq, tk, tv;
  const uint64_t rows = static_cast<uint64_t>(a.blocks) * a.Hkv * a.block;
  int rc = make_tmap_q(&tq, q, D, a.Hq, a.T, ldq * 2, a.G, a.q_rows);
  if (!rc) rc = rlb_make_tmap_2d(&tk, k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, D, rows, D * 2, 64, a.box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc) rc = rlb_make_tmap_2d(&tv, v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, D, rows, D * 2, 64, a.box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return -100 - rc;
  cudaError_t e = cudaFuncSetAttribute(tree_decode_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::SMEM);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int blocks = (a.max_rows + a.block_rows - 1) / a.block_rows;
  const dim3 grid = ctas ? dim3(ctas) : dim3(blocks, a.Hkv, a.B);
  e = rlb_launch_pdl(tree_decode_kernel<D>, grid, dim3(THREADS), Shape<D>::SMEM, stream, tq, tk, tv, a);
  if (e != cudaSuccess || !ctas) return static_cast<int>(e);
  return static_cast<int>(rlb_launch_pdl(tree_join_kernel<D>, dim3((a.part_rows + JOIN_ROWS - 1) / JOIN_ROWS, ctas), dim3(JOIN_ROWS * D / 8), 0, stream, a));
}
}  // namespace

// ctas > 0: so many CTAs share all tiles, at least `least` each, in groups that have the same tiles, each a block of a sequence's rows (group: the blocks of max_rows rows; 1: blocks one after the
// other); part_o [2 ctas, part_rows, D] and part_ml [2 ctas, part_rows, 2] fp32 with part_rows = min(max_rows, 128 / G) * G, on 32 bytes,
// cuts 32 bytes for each CTA.
// ctas 0: a CTA for each unit. q: rows on 16 bytes.
RLB_API int rlb_tree_decode(const void* q, long long ldq, const void* k, const void* v, int blocks, int block, const int* table, long long table_ld, int pages,
                            const int* ctx, const int* cu, int B, int T, int max_rows, int Hq, int Hkv, int D, const int* masks, long long masks_ld,
                            const int* positions, int window, float scale, int ctas, int group, int least, float* part_o, float* part_ml, void* cuts, void* out, long long ldo, int* status,
                            void* stream) {
  if (D != 64 && D != 128) return -2;
  if (Hkv < 1 || Hkv > 65535 || Hq % Hkv || Hq / Hkv > M_ROWS || B > 65535 || block < 16 || block % 16 || max_rows < 1 || max_rows > 256 || ldq % 8 || least < 1 || group < 1 || (ctas && ctas % group)) return -2;
  if (static_cast<long long>(blocks) * Hkv * block >= 0x7fffffffll || (ctas && (!part_o || !part_ml || !cuts))) return -2;
  TreeArgs a;
  a.blocks = blocks;
  a.block = block;
  a.pages = pages;
  a.block_shift = -1;
  for (int i = 4; i < 31; ++i)
    if (block == 1 << i) a.block_shift = i;
  a.box = block % 64 == 0 ? 64 : block % 32 == 0 ? 32 : 16;
  a.table = table;
  a.table_ld = table_ld;
  a.ctx = ctx;
  a.cu = cu;
  a.B = B;
  a.T = T;
  a.max_rows = max_rows;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.block_rows = M_ROWS / a.G;
  a.block_inv = 65536 / a.block_rows + 1;
  a.group_inv = 65536 / a.G + 1;
  a.q_rows = a.block_rows < max_rows ? a.block_rows : max_rows;
  a.masks = masks;
  a.masks_ld = masks_ld;
  a.positions = positions;
  a.window = window;
  // (hidden scores are infinite: they must not meet a factor of zero)
  a.scale_log2 = fabsf(scale) < 1e-30f ? copysignf(1e-30f, scale) : scale * LOG2E_F;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ldo = ldo;
  a.vec = ldo % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0;
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.part_o = ctas ? part_o : nullptr;
  a.part_ml = reinterpret_cast<float2*>(part_ml);
  a.part_rows = a.q_rows * a.G;
  a.cuts = static_cast<Cut*>(cuts);
  a.least = least;
  a.group = ctas ? group : 1;
  // (more units than run at once: 64 trees of 17 rows on ragged contexts to 1280 55 -> 52 us; where all have 804 tokens 46 -> 49)
  a.sorted = !ctas && B > 1 && B <= THREADS && static_cast<long long>(B) * Hkv * ((max_rows + a.block_rows - 1) / a.block_rows) > 2 * 148;
  a.status = status;
  return D == 64 ? launch<64>(q, ldq, k, v, a, ctas, static_cast<cudaStream_t>(stream)) : launch<128>(q, ldq, k, v, a, ctas, static_cast<cudaStream_t>(stream));
}
