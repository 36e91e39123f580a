// What the kernels of attention for drafted tokens share: their arguments, the division of the work among the blocks, and
// which keys a row sees.
//
// An entry e has q_len tokens (cu_q) and kv_len keys in its pages, the last q_len of them the tokens' own; start = kv_len -
// q_len keys are committed.  The row of token i and head h sees
//     a committed key j < start       iff there is no window, or j > positions[token] - window
//     the key start + k of token k    iff bit k % 32 of mask[token][k / 32] is set
// and nothing else; o = sum_j softmax_j(scale q . k_j) v_j over what it sees, zeros where it sees nothing.
//
// Division.  A unit is (entry, KV head, block of ROWS rows), a row being (token, head of the KV head's group); it walks its
// entry's keys in tiles of KEYS from the first one that the window leaves anybody.  All units' tiles stand in one list, in the
// order of entries, KV heads, blocks of rows; block c of C takes the tiles [c W / C, (c + 1) W / C) of the W, whatever units
// they belong to: every SM has the same number of tiles to within one, for one long request as for many ragged ones, and the
// division needs nothing from the host (lengths may change between replays of a graph).  A unit whose tiles lie with one
// block is written by that block; one that several share is left as unnormalised sums with their reference maximum and sum of
// weights (a slab per block: it has at most one unit that began before it and one that goes on behind it), which
// tree_merge_kernel adds in the order of the keys.  The sums depend on the lengths and C alone.
#pragma once

#include <math_constants.h>

#include "common.cuh"

namespace srlm {
namespace tree {

enum ErrorCode : int { ERR_PAGE = 71, ERR_ENTRY = 72 };

struct Args {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* out;
  const int* block_table;
  int table_stride;
  const int* cu_q;
  const int* kv_lens;
  const int* mask;
  int words;                 // of a token's mask
  int max_q_len;             // no entry has more tokens
  const int* positions;      // null without a window
  int n, T;                  // entries; rows of q and out
  int nq, nkv, hd, page_size;
  int num_pages;
  float scale_log2;          // score scale times log2(e)
  int window;
  int least_tiles;           // a block takes at least so many tiles
  int* err_flag;
  float* part_o;             // [2 C][ROWS][hd]
  float* part_ml;            // [2 C][ROWS][2]: reference maximum (log2 units), sum of weights
};

struct Entry {
  int q0, q_len, kv_len, start;
  int first_tile, tiles;     // key tiles that some row may see
  int blocks;                // of rows
};

// The entry's sizes; no tiles where there is nothing to do or the lengths contradict one another (FLAG: the error word is raised).
template <int ROWS, int KEYS>
__device__ __forceinline__ Entry entry_of(const Args& a, int e, bool flag = false) {
  Entry x;
  x.q0 = a.cu_q[e];
  x.q_len = a.cu_q[e + 1] - x.q0;
  x.kv_len = a.kv_lens[e];
  x.start = x.kv_len - x.q_len;
  const bool good = x.q_len >= 0 && x.q0 >= 0 && x.q0 + x.q_len <= a.T && x.start >= 0 && x.q_len <= a.max_q_len &&
                    x.kv_len <= (long long)a.table_stride * a.page_size;
  if (!good || x.q_len == 0) {
    if (!good && flag) atomicExch(a.err_flag, ERR_ENTRY);
    x.q_len = x.tiles = x.blocks = x.first_tile = 0;
    return x;
  }
  // no row's position is below start
  const int first = a.window > 0 ? max(0, x.start - a.window + 1) : 0;
  x.first_tile = first / KEYS;
  x.tiles = (x.kv_len + KEYS - 1) / KEYS - x.first_tile;
  x.blocks = (x.q_len * (a.nq / a.nkv) + ROWS - 1) / ROWS;
  return x;
}

__device__ __forceinline__ long long warp_total(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a block does in one go: tiles of one unit.
struct Piece {
  Entry x;
  int e, kvh, block;
  int tile_lo, tile_hi;        // tiles of the entry's keys, from its first key on
  bool begins, ends;           // the unit's first tile, its last one, are the piece's
};

// A block's share of the list.  Every warp that calls next() walks the same pieces.
template <int ROWS, int KEYS>
struct Walk {
  long long total, at, end;    // tiles of the list; the next one and the share's end
  int blocks;                  // blocks that have a share
  int e;                       // entry of the tile `at`, whose list begins at `base`
  long long base;
  Entry x;

  __device__ __forceinline__ long long weight(const Args& a, const Entry& y) const { return (long long)y.tiles * y.blocks * a.nkv; }

  // All lanes of a warp.  share: which of `blocks_there`; the entries' tiles are counted by the warp, 32 entries a turn.
  __device__ __forceinline__ void init(const Args& a, int share, int blocks_there, bool flag) {
    const int lane = threadIdx.x & 31;
    total = 0;
    for (int e0 = 0; e0 < a.n; e0 += 32)
      total += warp_total(e0 + lane < a.n ? weight(a, entry_of<ROWS, KEYS>(a, e0 + lane, flag)) : 0);
    const long long most = (total + a.least_tiles - 1) / a.least_tiles;
    blocks = (int)(most < blocks_there ? most : blocks_there);
    at = end = base = 0;
    e = 0;
    if (share < blocks) {
      at = share * total / blocks;
      end = (share + 1ll) * total / blocks;
    }
    if (at < end) seek(a, at);
  }
  // the entry that holds the tile `pos`
  __device__ __forceinline__ void seek(const Args& a, long long pos) {
    const int lane = threadIdx.x & 31;
    long long before = 0;
    for (int e0 = 0; e0 < a.n; e0 += 32) {
      const long long w = e0 + lane < a.n ? weight(a, entry_of<ROWS, KEYS>(a, e0 + lane)) : 0;
      long long upto = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned beyond = __ballot_sync(0xffffffffu, before + upto > pos);
      if (beyond) {
        const int l = __ffs(beyond) - 1;
        e = e0 + l;
        base = before + __shfl_sync(0xffffffffu, upto - w, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    x = entry_of<ROWS, KEYS>(a, e);
  }
  __device__ __forceinline__ bool next(const Args& a, Piece& p) {
    if (at >= end) return false;
    while (at - base >= weight(a, x)) {
      base += weight(a, x);
      x = entry_of<ROWS, KEYS>(a, ++e);          // (at is below the total: such an entry is there)
    }
    const long long unit = (at - base) / x.tiles;
    const int t = (int)(at - base - unit * x.tiles);
    const long long left = end - at;
    const int count = left < x.tiles - t ? (int)left : x.tiles - t;
    p.x = x;
    p.e = e;
    p.kvh = (int)(unit / x.blocks);
    p.block = (int)(unit % x.blocks);
    p.tile_lo = x.first_tile + t;
    p.tile_hi = p.tile_lo + count;
    p.begins = t == 0;
    p.ends = t + count == x.tiles;
    at += count;
    return true;
  }
};

// The slab of a piece that is not a whole unit.
__device__ __forceinline__ size_t slab_of(int share, bool begins) { return 2 * (size_t)share + (begins ? 1 : 0); }

// Which of the 32 keys from j0 on a row sees, as bits.  row_mask: the row's token's words; lo: its first committed key.
__device__ __forceinline__ uint32_t seen_bits(const Args& a, const int* row_mask, int j0, int start, int kv_len, int lo) {
  uint32_t bits = 0;
  if (j0 < start) {                               // committed keys [max(lo, j0), min(start, j0 + 32))
    const int from = max(lo - j0, 0), to = min(start - j0, 32);
    if (from < to) bits = (to >= 32 ? 0xffffffffu : (1u << to) - 1u) & ~(from > 0 ? (1u << from) - 1u : 0u);
  }
  const int k = j0 - start;                       // drafted tokens k, k + 1, ...
  if (k > -32) {
    uint32_t own;
    if (k < 0) {
      own = (uint32_t)row_mask[0] << -k;
    } else {
      const int w = k >> 5;
      const uint32_t low = w < a.words ? (uint32_t)row_mask[w] : 0u, high = w + 1 < a.words ? (uint32_t)row_mask[w + 1] : 0u;
      own = __funnelshift_r(low, high, k & 31);
    }
    const int to = min(kv_len - j0, 32);          // bits of tokens that the entry does not have are nobody's
    bits |= to <= 0 ? 0u : to >= 32 ? own : own & ((1u << to) - 1u);
  }
  return bits;
}

// The first committed key that a token's window leaves it (a position in front of the token's own place counts as that place).
__device__ __forceinline__ int first_key_of(const Args& a, int token, int start) {
  return a.window > 0 ? max(0, max(a.positions[token], start) - a.window + 1) : 0;
}

// The flat row of key j of KV head kvh in the pools [pages, kv heads, page size, head size]; a page that is not in the pool
// raises the error word and is read as page 0.
__device__ __forceinline__ long long row_of_key(const Args& a, const int* table, int j, int kvh) {
  const int pg = j / a.page_size;
  int page = table[pg];
  if (page < 0 || page >= a.num_pages) {
    atomicExch(a.err_flag, ERR_PAGE);
    page = 0;
  }
  return ((long long)page * a.nkv + kvh) * a.page_size + (j - pg * a.page_size);
}

// Values that are no numbers, in tiles where rows see different keys.  A product multiplies a value that a row does not see by
// zero, which leaves nothing of a finite one alone: such values are taken out of the tile (take_loose: eight bfloat16 numbers;
// whether there was one) and the rows that see them get them back as they are written (loose_values).
__device__ __forceinline__ bool take_loose(uint4& v) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  bool here = false;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bool lo = (w[k] & 0x7f80u) == 0x7f80u, hi = (w[k] & 0x7f800000u) == 0x7f800000u;
    if (lo) w[k] &= 0xffff0000u;
    if (hi) w[k] &= 0xffffu;
    here |= lo || hi;
  }
  return here;
}

// The sum of the non-finite values of dimension d that a row sees in the piece's masked tiles (all tiles are looked through: this is
// for rows whose cache holds such values).
template <int KEYS>
__device__ __noinline__ float loose_values(const Args& a, int start, int kv_len, const int* table, int kvh, int token, int d, int tile_lo,
                                           int tile_hi) {
  float sum = 0.f;
  const int lo = first_key_of(a, token, start);
  const bf16* v = (const bf16*)a.v_cache;
  for (int j0 = tile_lo * KEYS; j0 < tile_hi * KEYS && j0 < kv_len; j0 += 32) {
    if (j0 / KEYS * KEYS + KEYS <= start && (a.window <= 0 || j0 / KEYS * KEYS >= kv_len - a.window)) continue;
    uint32_t bits = seen_bits(a, a.mask + (size_t)token * a.words, j0, start, kv_len, lo);
    while (bits) {
      const int j = j0 + __ffs(bits) - 1;
      bits &= bits - 1;
      const float f = to_float(v[row_of_key(a, table, j, kvh) * a.hd + d]);
      if (!isfinite(f)) sum += f;
    }
  }
  return sum;
}

// Adds the slabs of the unit that begins in share blockIdx.x and goes on behind it, eight rows a block, a warp a row, a lane
// every 32nd dimension: out = sum_z O_z 2^(m_z - M) / sum_z l_z 2^(m_z - M), M the largest reference of a slab that saw a key.
template <typename T, int ROWS, int KEYS>
__global__ void __launch_bounds__(256) tree_merge_kernel(const __grid_constant__ Args a, int blocks_there) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = blockIdx.x;
  Walk<ROWS, KEYS> w;
  w.init(a, share, blocks_there, false);
  if (w.at >= w.end) return;
  const long long lo = w.at, last = w.end - 1;
  w.seek(a, last);
  const long long unit = (last - w.base) / w.x.tiles, from = w.base + unit * w.x.tiles, to = from + w.x.tiles;
  if (from < lo || to <= w.end) return;                        // another share's unit, or a whole one
  const int kvh = (int)(unit / w.x.blocks), block = (int)(unit % w.x.blocks), g = a.nq / a.nkv;
  const int row = blockIdx.y * 8 + warp, r = block * ROWS + row;
  if (row >= ROWS || r >= w.x.q_len * g) return;
  const int share_last = (int)((to * w.blocks - 1) / w.total);  // whose tiles hold the unit's last one
  float M = -CUDART_INF_F;
  for (int s = share + lane; s <= share_last; s += 32) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (slab_of(s, s == share) * ROWS + row) * 2);
    if (ml.y > 0.f) M = fmaxf(M, ml.x);
  }
  M = warp_max(M);
  constexpr int MOST = 8;                                       // dimensions of a lane: heads up to 256
  float acc[MOST], L = 0.f;
#pragma unroll
  for (int i = 0; i < MOST; ++i) acc[i] = 0.f;
  for (int s = share; s <= share_last; ++s) {
    const size_t at = slab_of(s, s == share) * ROWS + row;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
    if (!(ml.y > 0.f)) {
      if (ml.y != ml.y) L = ml.y;                               // a score that was no number
      continue;
    }
    const float wz = exp2f(ml.x - M);
    L += wz * ml.y;
    if (wz > 0.f) {
#pragma unroll
      for (int i = 0; i < MOST; ++i)
        if (lane + 32 * i < a.hd) acc[i] += wz * a.part_o[at * a.hd + lane + 32 * i];
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* dst = (T*)a.out + ((size_t)(w.x.q0 + r / g) * a.nq + kvh * g + r % g) * a.hd;
#pragma unroll
  for (int i = 0; i < MOST; ++i)
    if (lane + 32 * i < a.hd) dst[lane + 32 * i] = from_float<T>(acc[i] * inv);
}

// The forms.  Each gives its blocks (C) and rows of a unit, which size the slabs.
struct Form {
  int blocks, rows;
};
Form simt_form(int hd, int sms);
int run_simt(const Args& a, int dtype, int max_rows, int sms, cudaStream_t stream);
bool mma_takes(int hd);                            // bfloat16
Form mma_form(int hd, int max_rows, int sms);
int run_mma(const Args& a, int max_rows, int sms, cudaStream_t stream);
bool tcgen05_takes(int hd, int page_size);         // bfloat16
Form tcgen05_form(int sms);
int run_tcgen05(const Args& a, int max_rows, int sms, cudaStream_t stream);

}  // namespace tree
}  // namespace srlm
