// What the kernels of attention for drafted tokens share: their arguments, the division of the work among the blocks, and
// which keys a row sees.
//
// An entry e has q_len tokens (cu_q) and kv_len keys in its pages, the last q_len of them the tokens' own; start = kv_len -
// q_len keys are committed.  The row of token i and head h sees
//     a committed key j < start       iff there is no window, or j > positions[token] - window, start <= positions[token] < kv_len
//     the key start + k of token k    iff bit k % 32 of mask[token][k / 32] is set
// and nothing else; o = sum_j softmax_j(scale q . k_j) v_j over what it sees, zeros where it sees nothing.
//
// Division.  A unit is (entry, KV head, block of ROWS rows), a row being (token, head of the KV head's group); it walks its
// entry's keys in tiles of KEYS from the first one that the window leaves anybody.  All units' tiles stand in one list, in the
// order of entries, KV heads, blocks of rows; share c of C is the tiles [c W / C, (c + 1) W / C) of the W, whatever units
// they belong to: every SM has the same number of tiles to within one, for one long request as for many ragged ones, and the
// division needs nothing from the host (lengths may change between replays of a graph).  A unit whose tiles lie with one
// block is written by that block; one that several share is left as unnormalised sums with their reference maximum and sum of
// weights (a slab per block: it has at most one unit that began before it and one that goes on behind it), which
// tree_merge_kernel adds in the order of the keys.  The sums depend on the lengths and C alone.
// Small work is divided along the units instead: each into as many equal parts as keep every block at one part.  A block whose
// share reaches into a second unit begins anew with its rows and its first keys and leaves two slabs, which costs it more than
// SPARE_TILES tiles (entries of 128 rows, 8 KV heads of 128, us, shares of all tiles | parts: 1 behind 600 keys 22.1 | 15.8, 8
// behind 2,000 29.9 | 25.8, 16 behind 2,000 51.5 | 34.7, 16 behind 4,000 68.1 | 56.0, 12 behind 8,000 77.0 | 82.5, which is beyond
// the 12 spare tiles).
// More units than blocks are dealt out whole where that is no longer, a beginning and the merge counted as BEGIN_TILES tiles each
// (entries of 64 rows, us, shares of all tiles | whole units: 32 behind 600 keys 41.5 | 30.6, 64 behind 1,000 75.4 | 68.0; 20 behind
// 2,000, two rounds of 17 tiles, 47.9 | 55.8).
// Where units of several blocks of rows read more keys than the L2 cache holds, their blocks go through the same tiles at the same
// time, as many thread blocks side by side as the units have blocks of rows (members): the keys come from memory once and not once
// for each (8 entries behind 12,000 to 24,000 keys, 8 KV heads of 128, us, apart | side by side: 320 rows 273 | 237; behind 8,000 to
// 16,000, 512 rows 263 | 212, 256 rows 141 | 122; 256 rows behind 4,000, which the cache holds, 59.7 | 58.5).
#pragma once

#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace srlm {
namespace tree {

enum ErrorCode : int { ERR_PAGE = 71, ERR_ENTRY = 72, ERR_POSITION = 75 };

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
  int nq, nkv, g, hd, page_size;      // g: query heads of a KV head
  int num_pages;
  float scale_log2;          // score scale times log2(e)
  float key_bytes;           // of a key and its value in one KV head
  int window;
  int least_tiles;           // a block takes at least so many tiles
  int* err_flag;
  float* part_o;             // slabs [2 C][hd][ROWS]: neighbouring rows side by side, as the threads that write and read them are
  float* part_ml;            // [2 C][ROWS][2]: reference maximum (log2 units), sum of weights
  int4* part_units;          // [C]: the unit that begins in share C and goes on behind it: its slabs (0: none such) | members << 16, first row
                             // of its entry's rows, first token of the entry, KV head | rows << 16
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
  const int q1 = a.cu_q[e + 1];
  x.kv_len = a.kv_lens[e];
  // compared before they are subtracted: a difference of wild numbers may pass 32 bits and look right again
  const bool rows = x.q0 >= 0 && q1 >= x.q0 && q1 <= a.T;
  x.q_len = rows ? q1 - x.q0 : 0;
  const bool good = rows && x.q_len <= a.max_q_len && x.kv_len >= x.q_len &&
                    x.kv_len <= (long long)a.table_stride * a.page_size;
  if (!good || x.q_len == 0) {
    if (!good && flag) atomicExch(a.err_flag, ERR_ENTRY);
    x.q_len = x.start = x.tiles = x.blocks = x.first_tile = 0;
    return x;
  }
  x.start = x.kv_len - x.q_len;
  // no row's position is below start
  const int first = a.window > 0 ? max(0, x.start - a.window + 1) : 0;
  x.first_tile = first / KEYS;
  x.tiles = (x.kv_len + KEYS - 1) / KEYS - x.first_tile;
  x.blocks = (x.q_len * a.g + ROWS - 1) / ROWS;
  return x;
}

// What a block does in one go: tiles of one unit.
struct Piece {
  Entry x;
  int e, kvh, block;
  int tile_lo, tile_hi;        // tiles of the entry's keys, from its first key on
  bool begins, ends;           // the unit's first tile, its last one, are the piece's
};

constexpr int SPARE_TILES = 12, BEGIN_TILES = 10;
constexpr float L2_HELD = 64e6f;     // bytes of keys and values that units read one behind another still find in the L2 cache

// A block's share of the list.  Every warp that calls next() walks the same pieces.  (A list is shorter than 2^31: the entry
// point sees to it.)
template <int ROWS, int KEYS>
struct Walk {
  int at, end;                 // the next tile and the share's end
  int members, member;         // thread blocks side by side on a share, each with a block of rows; 1: shares of all units' tiles;
                               // 0: of whole units, and what counts tiles here counts units
  int each, more;              // tiles of a share; the first `more` shares have one more
  int e, base;                 // entry of the tile `at`, whose list begins at `base`
  int parts;                   // 0, or of how many parts of its unit this block has one: `at` the unit, `base` the part
  Entry x;

  __device__ __forceinline__ int weight(const Args& a, const Entry& y) const {
    return a.nkv * (members > 1 ? y.tiles : members == 1 ? y.tiles * y.blocks : y.blocks);
  }
  __device__ __forceinline__ int first_of(int share) const { return share * each + min(share, more); }
  // the share that holds the tile `pos`
  __device__ __forceinline__ int share_of(int pos) const {
    const int longer = more * (each + 1);
    return pos < longer ? pos / (each + 1) : more + (pos - longer) / each;
  }

  // All lanes of a warp: the entries' tiles are counted by the warp, 32 entries a turn.
  __device__ __forceinline__ void init(const Args& a, bool flag) {
    const int lane = threadIdx.x & 31, there = gridDim.x;
    Entry mine;
    int whole = 0, single = 0, most = 0, units = 0, longest = 0;      // tiles of all units, of one block of rows each; most blocks of
                                                 // rows; units, and most tiles of one
    for (int e0 = 0; e0 < a.n; e0 += 32) {
      if (e0 + lane < a.n) mine = entry_of<ROWS, KEYS>(a, e0 + lane, flag);
      else mine.tiles = mine.blocks = 0;
      const int w = mine.tiles * a.nkv;
      single += __reduce_add_sync(0xffffffffu, w);
      whole += __reduce_add_sync(0xffffffffu, w * mine.blocks);
      most = max(most, __reduce_max_sync(0xffffffffu, mine.blocks));
      units += __reduce_add_sync(0xffffffffu, mine.blocks * a.nkv);
      longest = max(longest, __reduce_max_sync(0xffffffffu, mine.tiles));
    }
    members = 1;
    parts = 0;
    if (a.n <= 32 && whole > 0) {
      const int own = mine.blocks * a.nkv;
      const int least = max(a.least_tiles, (whole + there - 1) / there);
      for (int tiles = least; tiles <= least + SPARE_TILES; ++tiles) {
        const int each_unit = (mine.tiles + tiles - 1) / tiles, blocks = own * each_unit;
        if ((int)__reduce_add_sync(0xffffffffu, blocks) > there) continue;
        int upto = blocks;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const unsigned beyond = __ballot_sync(0xffffffffu, upto > (int)blockIdx.x);
        at = end = base = 0;
        if (!beyond) return;                     // (more blocks than parts)
        e = __ffs(beyond) - 1;
        parts = __shfl_sync(0xffffffffu, each_unit, e);
        const int place = blockIdx.x - __shfl_sync(0xffffffffu, upto - blocks, e);
        at = place / parts;
        base = place - at * parts;
        end = at + 1;
        x = entry_of<ROWS, KEYS>(a, e);
        return;
      }
    }
    if (most > 1 && most <= 8 && (float)single * KEYS * a.key_bytes > L2_HELD) {
      // side by side, unless blocks of rows that some entries do not have would leave a tenth of the time empty
      const int used = there / most * most;
      if ((float)whole * there >= 0.9f * (float)single * most * used && (float)whole >= 0.9f * (float)single * most) members = most;
    }
    if (members == 1) {
      // whole units, where the longest share of them is no longer than tiles, beginnings and the merge of shares of tiles
      const float rounds = (units + there - 1) / there;
      if (rounds * (longest + BEGIN_TILES) < (float)whole / there + BEGIN_TILES * ((float)units / there + 2.f)) members = 0;
    }
    const int total = members > 1 ? single : members == 1 ? whole : units;
    const int share = members > 1 ? blockIdx.x / members : blockIdx.x;
    member = members > 1 ? blockIdx.x - share * members : 0;
    const int shares = members > 0 ? min((total + a.least_tiles - 1) / a.least_tiles, there / members) : min(total, there);
    at = end = base = e = each = more = 0;
    if (share >= shares) return;
    each = total / shares;
    more = total - each * shares;
    at = first_of(share);
    end = first_of(share + 1);
    // the entry that holds the tile
    int before = 0;
    for (int e0 = 0; e0 < a.n; e0 += 32) {
      if (a.n > 32) {
        if (e0 + lane < a.n) mine = entry_of<ROWS, KEYS>(a, e0 + lane);
        else mine.tiles = mine.blocks = 0;
      }
      const int w = weight(a, mine);
      int upto = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned beyond = __ballot_sync(0xffffffffu, before + upto > at);
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
    if (parts > 0) {
      if (at >= end) return false;
      p.x = x;
      p.e = e;
      p.kvh = at / x.blocks;
      p.block = at - p.kvh * x.blocks;
      // the first `longer` parts have a tile more (no product of parts and tiles: it would pass 32 bits)
      const int part = x.tiles / parts, longer = x.tiles - part * parts;
      p.tile_lo = x.first_tile + base * part + min(base, longer);
      p.tile_hi = p.tile_lo + part + (base < longer ? 1 : 0);
      p.begins = base == 0;
      p.ends = base + 1 == parts;
      at = end;
      return true;
    }
    while (at < end) {
      while (at - base >= weight(a, x)) {
        base += weight(a, x);
        x = entry_of<ROWS, KEYS>(a, ++e);        // (at is below the total: such an entry is there)
      }
      int unit, t = 0, count = x.tiles;
      if (members > 0) {
        unit = (at - base) / x.tiles;
        t = at - base - unit * x.tiles;
        count = min(end - at, x.tiles - t);
        at += count;
      } else {
        unit = at++ - base;
      }
      if (member >= x.blocks) continue;          // a block of rows that this entry does not have
      p.x = x;
      p.e = e;
      p.kvh = members > 1 ? unit : unit / x.blocks;
      p.block = members > 1 ? member : unit - p.kvh * x.blocks;
      p.tile_lo = x.first_tile + t;
      p.tile_hi = p.tile_lo + count;
      p.begins = t == 0;
      p.ends = t + count == x.tiles;
      return true;
    }
    return false;
  }
};

// The slab of a block's piece that is not a whole unit.
__device__ __forceinline__ size_t slab_of(int block, bool begins) { return 2 * (size_t)block + (begins ? 1 : 0); }

// Which keys of a tile a row sees, as bits, 32 a word.  words(): the part of the row's mask that the tile needs, N + 1 loads in
// flight at once, which may be made ahead; bits(): the tile's keys from j0 on.
template <int N>
struct Sight {
  uint32_t w[N + 1];
  __device__ __forceinline__ void words(const Args& a, int token, int j0, int start) {
    const int* row_mask = a.mask + (size_t)token * a.words;
    const int first = (j0 - start) >> 5;                         // (rounded down: below zero the tile begins in front of the tokens)
#pragma unroll
    for (int i = 0; i <= N; ++i) w[i] = first + i >= 0 && first + i < a.words ? (uint32_t)row_mask[first + i] : 0u;
  }
  // lo: the row's first committed key
  __device__ __forceinline__ void bits(uint32_t (&out)[N], int j0, int start, int kv_len, int lo) const {
    const int shift = (j0 - start) & 31;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = j0 + 32 * i;
      uint32_t own = __funnelshift_r(w[i], w[i + 1], shift);     // drafted tokens j - start, ...
      const int to = kv_len - j;                                 // bits of tokens that the entry does not have are nobody's
      own = to <= 0 ? 0u : to >= 32 ? own : own & ((1u << to) - 1u);
      const int from = max(lo - j, 0), upto = min(start - j, 32);      // committed keys [max(lo, j), min(start, j + 32))
      if (from < upto) own |= (upto >= 32 ? 0xffffffffu : (1u << upto) - 1u) & ~((1u << from) - 1u);
      out[i] = own;
    }
  }
};

// The first committed key that a token's window leaves it.  A position outside [start, kv_len) is none of the entry's: it raises the
// error word and counts as the nearest of them.  (Which tiles every row sees whole, and which the entry needs at all, is decided by those
// two bounds; the entry's last tile is never one of the former, so each row comes by here.)
__device__ __forceinline__ int first_key_of(const Args& a, int token, int start, int kv_len) {
  if (a.window <= 0) return 0;
  const int given = a.positions[token], position = min(max(given, start), kv_len - 1);
  if (position != given) atomicExch(a.err_flag, ERR_POSITION);
  return max(0, position - a.window + 1);
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
// zero, which leaves nothing of a finite one alone: such values are taken out of the tile (take_loose: eight bfloat16 numbers or four
// float32 ones; whether there was one) and the rows that see them get them back as they are written (loose_values).
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

__device__ __forceinline__ bool take_loose(float4& v) {
  bool here = false;
  float* f = reinterpret_cast<float*>(&v);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (!isfinite(f[k])) {
      f[k] = 0.f;
      here = true;
    }
  return here;
}

// The sum of the non-finite values of dimension d that a row sees in the piece's masked tiles (all tiles are looked through: this is
// for rows whose cache holds such values).
template <typename T, int KEYS>
__device__ __noinline__ float loose_values(const Args& a, int start, int kv_len, const int* table, int kvh, int token, int d, int tile_lo,
                                           int tile_hi) {
  float sum = 0.f;
  const int lo = first_key_of(a, token, start, kv_len);
  const T* v = (const T*)a.v_cache;
  for (int j0 = tile_lo * KEYS; j0 < tile_hi * KEYS && j0 < kv_len; j0 += 32) {
    if (j0 / KEYS * KEYS + KEYS <= start && (a.window <= 0 || j0 / KEYS * KEYS >= kv_len - a.window)) continue;
    Sight<1> sight;
    uint32_t bits[1];
    sight.words(a, token, j0, start);
    sight.bits(bits, j0, start, kv_len, lo);
    while (bits[0]) {
      const int j = j0 + __ffs(bits[0]) - 1;
      bits[0] &= bits[0] - 1;
      const float f = to_float(v[row_of_key(a, table, j, kvh) * a.hd + d]);
      if (!isfinite(f)) sum += f;
    }
  }
  return sum;
}

// What a block leaves for the merge beside its slabs, by one thread: the unit that goes on behind its share, or that there is none.
__device__ __forceinline__ void leave_no_unit(const Args& a) { a.part_units[blockIdx.x] = make_int4(0, 0, 0, 0); }
template <int ROWS, int KEYS>
__device__ __forceinline__ void leave_unit(const Args& a, const Walk<ROWS, KEYS>& w, const Piece& p) {
  if (!p.begins || p.ends) return;
  const int to = w.at + (p.x.first_tile + p.x.tiles - p.tile_hi), r0 = p.block * ROWS;
  const int slabs = w.parts > 0 ? w.parts : w.share_of(to - 1) - blockIdx.x / w.members + 1;
  a.part_units[blockIdx.x] = make_int4(slabs | w.members << 16, r0, p.x.q0,
                                       p.kvh | min(ROWS, p.x.q_len * a.g - r0) << 16);
}

// Adds the slabs of the unit that begins in block blockIdx.x's share and goes on behind it: out = sum_z O_z 2^(m_z - M) / sum_z l_z
// 2^(m_z - M), M the largest reference of a slab that saw a key; which slabs a warp adds depends on their number alone.
// A block has 32 rows (blockIdx.y), a lane one of them and MERGE_DIMS dimensions (of units of fewer rows a warp has several such runs);
// what warps the dimensions leave deal the slabs among themselves and add up in shared memory.  The kernel is all latency: the
// unit's record, the slabs, the result, one behind another, in a launch of its own.  It adds 7 to 9 us to a call whose units are divided
// (ten calls in a graph, us, with | without it: 24 tokens of 32 heads behind 16,000 keys 25.7 | 17.1, 8 entries of 20 to 32 behind 1,000
// to 3,000 27.7 | 20.6, 6 of up to 40 over heads of 64 under a window of 1,000 22.7 | 13.5, 3 of up to 12 in float32 29.3 | 22.0), and
// nothing that shows to the largest (8 entries of 64 behind 16,000 to 32,768, 40 heads, 295 | 297).
constexpr int MERGE_WARPS = 32, MERGE_DIMS = 8, MERGE_TURNS = 4;

template <typename T, int ROWS>
__global__ void __launch_bounds__(32 * MERGE_WARPS) tree_merge_kernel(const __grid_constant__ Args a, int dim_warps, int turns) {
  constexpr int RL = ROWS < 32 ? ROWS : 32;
  __shared__ float acc_sh[(MERGE_WARPS - MERGE_WARPS / MERGE_TURNS) * MERGE_DIMS][32];
  __shared__ float2 ml_sh[MERGE_WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int turn = warp / dim_warps, share = blockIdx.x, row = blockIdx.y * RL + lane % RL;
  const int d0 = (warp % dim_warps * (32 / RL) + lane / RL) * MERGE_DIMS, dims = min(MERGE_DIMS, a.hd - d0);
  pdl_wait();
  pdl_trigger();
  const int4 unit = a.part_units[share];
  const int slabs = unit.x & 0xffff, members = unit.x >> 16, kvh = unit.w & 0xffff, rows = unit.w >> 16;
  if (slabs == 0 || (int)blockIdx.y * RL >= rows) return;
  float acc[MERGE_DIMS], M = -CUDART_INF_F, L = 0.f;
#pragma unroll
  for (int i = 0; i < MERGE_DIMS; ++i) acc[i] = 0.f;
  constexpr int AHEAD = 2;                                           // slabs in flight (four: 2 us more, for their code)
  for (int z0 = row < rows ? turn : slabs; z0 < slabs; z0 += AHEAD * turns) {
    float2 v[AHEAD];
    float o[AHEAD][MERGE_DIMS];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int z = z0 + k * turns;
      const size_t slab = slab_of(share + z * members, z == 0);
      const float* src = a.part_o + (slab * a.hd + d0) * ROWS + row;
      v[k] = z < slabs ? *reinterpret_cast<const float2*>(a.part_ml + (slab * ROWS + row) * 2) : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < MERGE_DIMS; ++i) o[k][i] = z < slabs && i < dims ? src[i * ROWS] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (v[k].y > 0.f) {                                            // (a slab of no key holds nothing)
        const float m_new = fmaxf(M, v[k].x), f = exp2f(v[k].x - m_new), old = exp2f(M - m_new);
        M = m_new;
        L = L * old + f * v[k].y;
#pragma unroll
        for (int i = 0; i < MERGE_DIMS; ++i) acc[i] = acc[i] * old + f * o[k][i];
      } else if (v[k].y != v[k].y) {
        L = v[k].y;                                                  // (a score that was no number makes the row none)
      }
    }
  }
  if (turns > 1) {
    if (turn > 0) {
      ml_sh[warp][lane] = make_float2(M, L);
#pragma unroll
      for (int i = 0; i < MERGE_DIMS; ++i) acc_sh[(warp - dim_warps) * MERGE_DIMS + i][lane] = acc[i];
    }
    __syncthreads();
    if (turn > 0) return;
#pragma unroll 1
    for (int w = warp + dim_warps; w < turns * dim_warps; w += dim_warps) {
      const float2 v = ml_sh[w][lane];
      if (v.y > 0.f) {
        const float m_new = fmaxf(M, v.x), f = exp2f(v.x - m_new), old = exp2f(M - m_new);
        M = m_new;
        L = L * old + f * v.y;
#pragma unroll
        for (int i = 0; i < MERGE_DIMS; ++i) acc[i] = acc[i] * old + f * acc_sh[(w - dim_warps) * MERGE_DIMS + i][lane];
      } else if (v.y != v.y) {
        L = v.y;
      }
    }
  }
  if (row >= rows || dims <= 0) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int g = a.g, r = unit.y + row;
  T* dst = (T*)a.out + ((size_t)(unit.z + r / g) * a.nq + kvh * g + r % g) * a.hd + d0;
#pragma unroll
  for (int i = 0; i < MERGE_DIMS; ++i) acc[i] *= inv;
  if constexpr (sizeof(T) == 2) {
    if (a.hd % MERGE_DIMS == 0 && (uintptr_t)a.out % 16 == 0) {
      __nv_bfloat162 p[MERGE_DIMS / 2];
#pragma unroll
      for (int i = 0; i < MERGE_DIMS / 2; ++i) p[i] = __floats2bfloat162_rn(acc[2 * i], acc[2 * i + 1]);
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(p);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < MERGE_DIMS; ++i)
    if (i < dims) dst[i] = from_float<T>(acc[i]);
}
// Whether some unit can have several slabs.  None can where every unit has at most least_tiles tiles by the block table's width, and there
// are no more units than blocks (their parts are whole units then).
inline bool merges(const Args& a, int blocks, int rows, int keys) {
  const long long tiles = ((long long)a.table_stride * a.page_size + keys - 1) / keys;
  const long long units = (long long)a.n * a.nkv * ((a.max_q_len * a.g + rows - 1) / rows);
  return a.n > 32 || units > blocks || tiles > a.least_tiles;
}
template <typename T, int ROWS, int KEYS>
inline void launch_merge(const Args& a, int blocks, cudaStream_t stream) {
  if (!merges(a, blocks, ROWS, KEYS)) return;
  constexpr int RL = ROWS < 32 ? ROWS : 32, SPAN = 32 / RL * MERGE_DIMS;
  const int dim_warps = (a.hd + SPAN - 1) / SPAN, turns = std::min(MERGE_TURNS, MERGE_WARPS / dim_warps);
  const int max_rows = std::min(a.max_q_len * a.g, ROWS);
  launch_pdl(tree_merge_kernel<T, ROWS>, dim3(blocks, (max_rows + RL - 1) / RL), dim3(32 * dim_warps * turns), 0, stream, a, dim_warps, turns);
}

// Lets a kernel have `bytes` of shared memory, once a device (the attribute stays with the kernel; each kernel has a `have` of its own).
// The same number on every call of a kernel, the most that any of its calls takes: threads that come here together write the same.
inline cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<bool> (&have)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::atomic<bool>* slot = dev < 64 ? &have[dev] : nullptr;
  if (slot && slot->load(std::memory_order_relaxed)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && slot) slot->store(true, std::memory_order_relaxed);
  return e;
}

// The forms.  Each gives its blocks (C) and the rows of a unit, which size the slabs, and the keys of a tile.
struct Form {
  int blocks, rows, keys;
};
Form simt_form(int hd, int max_rows, int sms);
int run_simt(const Args& a, int dtype, int max_rows, int sms, cudaStream_t stream);
bool mma_takes(int hd);                            // bfloat16
Form mma_form(int hd, int max_rows, int sms);
int run_mma(const Args& a, int max_rows, int sms, cudaStream_t stream);
bool tcgen05_takes(int hd, int page_size);         // bfloat16
Form tcgen05_form(int sms);
int run_tcgen05(const Args& a, int sms, cudaStream_t stream);

}  // namespace tree
}  // namespace srlm
