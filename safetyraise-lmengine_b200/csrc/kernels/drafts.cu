// Drafted tokens around the attention that runs them, and pages of the cache: which tokens each sees, which are accepted, the
// accepted ones' rows moved together, pages copied.
#include <algorithm>
#include <vector>

#include "common.cuh"

namespace srlm {
namespace drafts {

enum ErrorCode : int { ERR_PARENT = 73, ERR_PATH = 74 };

// An entry's tokens, or -1 where its bounds are none of T rows: compared before they are subtracted, for a difference of wild
// numbers may pass 32 bits and look right again.
__device__ __forceinline__ int tokens_of(int q0, int q1, int T) { return q0 >= 0 && q1 >= q0 && q1 <= T ? q1 - q0 : -1; }

// ---------------------------------------------------------------------------
// positions[t] = committed tokens + depth of t, and bit k of mask[t]: k is t or one of its ancestors (at most window - 1 above
// it, where there is a window).  A thread a token: it goes up its line, whose numbers fall, and writes its words from the last
// to the first, each once.
// ---------------------------------------------------------------------------
constexpr int TREE_THREADS = 128;

__global__ void __launch_bounds__(TREE_THREADS) draft_tree_kernel(const int* __restrict__ parents, const int* __restrict__ cu_q,
                                                                  const int* __restrict__ kv_lens, int* __restrict__ positions,
                                                                  int* __restrict__ mask, int words, int T, int window,
                                                                  int* __restrict__ err) {
  pdl_wait();
  pdl_trigger();
  const int e = blockIdx.x;
  const int q0 = cu_q[e], q_len = tokens_of(q0, cu_q[e + 1], T), kv_len = kv_lens[e];
  if (q_len <= 0 || q_len > 32ll * words || kv_len < q_len) {
    if (q_len != 0 && threadIdx.x == 0) atomicExch(err, ERR_PARENT);
    return;
  }
  const int start = kv_len - q_len;
  const int* up = parents + q0;
  for (int i = blockIdx.y * TREE_THREADS + threadIdx.x; i < q_len; i += gridDim.y * TREE_THREADS) {
    int* row = mask + (size_t)(q0 + i) * words;
    int depth = 0, w = words - 1;
    uint32_t bits = 0;
    for (int k = i;;) {
      if (window <= 0 || depth < window) {
        for (; w > k >> 5; --w) {
          row[w] = (int)bits;
          bits = 0;
        }
        bits |= 1u << (k & 31);
      }
      const int p = up[k];
      if (p < 0 || p >= k) {                       // a root; a parent that does not stand before its child makes one too
        if (p != -1) atomicExch(err, ERR_PARENT);
        break;
      }
      k = p;
      ++depth;
    }
    for (; w >= 0; --w) {
      row[w] = (int)bits;
      bits = 0;
    }
    positions[q0 + i] = start + depth;
  }
}

// ---------------------------------------------------------------------------
// From each entry's token 0 on: the first child whose token is the target of the one before.  A warp an entry.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(32) accept_drafts_kernel(const int* __restrict__ tokens, const int* __restrict__ parents,
                                                           const int* __restrict__ targets, const int* __restrict__ cu_q, int T,
                                                           int* __restrict__ path, int cap, int* __restrict__ count,
                                                           int* __restrict__ next, int* __restrict__ err) {
  pdl_wait();
  pdl_trigger();
  const int e = blockIdx.x, lane = threadIdx.x;
  const int q0 = cu_q[e], q_len = tokens_of(q0, cu_q[e + 1], T);
  int* line = path + (size_t)e * cap;
  if (q_len <= 0) {
    if (lane == 0) {
      if (q_len != 0) atomicExch(err, ERR_PARENT);
      count[e] = 0;
      next[e] = -1;
    }
    for (int i = lane; i < cap; i += 32) line[i] = -1;
    return;
  }
  int at = 0, kept = 1;
  if (lane == 0) line[0] = 0;
  int want = targets[q0];
  while (kept < cap) {
    int child = -1;
    for (int k0 = at + 1; k0 < q_len; k0 += 32) {          // children stand behind their parent
      const int k = k0 + lane;
      const bool hit = k < q_len && parents[q0 + k] == at && tokens[q0 + k] == want;
      const unsigned who = __ballot_sync(0xffffffffu, hit);
      if (who) {
        child = k0 + __ffs(who) - 1;
        break;
      }
    }
    if (child < 0) break;
    at = child;
    want = targets[q0 + at];
    if (lane == 0) line[kept] = at;
    ++kept;
  }
  if (lane == 0) {
    count[e] = kept;
    next[e] = want;
  }
  for (int i = kept + lane; i < cap; i += 32) line[i] = -1;
}

// ---------------------------------------------------------------------------
// The accepted tokens' rows of the cache side by side: place start + i takes what place start + path[i] holds, in every slab
// (layer, keys or values) and KV head.  path rises and path[i] >= i, so a thread that owns some bytes of every row and takes
// the rows in order never reads a place that it has written: no second buffer, no barrier.
// ---------------------------------------------------------------------------
constexpr int KEEP_THREADS = 128, KEEP_ROWS = 64;          // rows whose places are found at a time

template <typename V>
__global__ void __launch_bounds__(KEEP_THREADS) keep_drafts_kernel(V* __restrict__ pool, const int* __restrict__ block_table,
                                                                   int table_stride, const int* __restrict__ cu_q,
                                                                   const int* __restrict__ kv_lens, const int* __restrict__ path,
                                                                   int cap, const int* __restrict__ count, int slabs,
                                                                   int num_pages, int nkv, int page_size, int row_pieces,
                                                                   int* __restrict__ err) {
  __shared__ long long from_sh[KEEP_ROWS], to_sh[KEEP_ROWS];      // rows of a slab's first head; -1: the move ends here
  pdl_wait();
  pdl_trigger();
  const int e = blockIdx.y;
  const int q_len = tokens_of(cu_q[e], cu_q[e + 1], 0x7fffffff), kv_len = kv_lens[e], kept = min(count[e], cap);
  const int* line = path + (size_t)e * cap;
  const int* table = block_table + (size_t)e * table_stride;
  const long long per_slab = (long long)nkv * row_pieces, columns = slabs * per_slab;
  const long long col = (long long)blockIdx.x * KEEP_THREADS + threadIdx.x;
  const long long slab = col / per_slab;
  const int in_slab = (int)(col - slab * per_slab), head = in_slab / row_pieces, piece = in_slab - head * row_pieces;
  V* base = pool + (slab * num_pages * nkv * page_size + (long long)head * page_size) * row_pieces + piece;
  for (int i0 = 0; i0 < kept; i0 += KEEP_ROWS) {
    const int rows = min(KEEP_ROWS, kept - i0);
    for (int i = threadIdx.x; i < rows; i += KEEP_THREADS) {
      const int k = line[i0 + i], before = i0 + i > 0 ? line[i0 + i - 1] : -1;
      long long at[2] = {-1, -1};
      bool good = q_len >= 0 && kv_len >= q_len && k >= i0 + i && k > before && k < q_len;
      for (int s = 0; s < 2 && good; ++s) {
        const int place = kv_len - q_len + (s ? i0 + i : k), pg = place / page_size;
        const int page = pg < table_stride ? table[pg] : -1;
        good = page >= 0 && page < num_pages;
        at[s] = ((long long)page * nkv * page_size + (place - pg * page_size)) * row_pieces;
      }
      if (!good) atomicExch(err, ERR_PATH);
      from_sh[i] = good ? at[0] : -1;
      to_sh[i] = at[1];
    }
    __syncthreads();
    bool end = false;
    if (col < columns) {
      constexpr int AHEAD = 8;
      for (int i = 0; i < rows && !end; i += AHEAD) {
        V v[AHEAD];
        int n = 0;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
          if (!end && i + j < rows) {
            if (from_sh[i + j] < 0) end = true;
            else if (from_sh[i + j] != to_sh[i + j]) v[j] = base[from_sh[i + j]], n = j + 1;
          }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
          if (j < n && from_sh[i + j] != to_sh[i + j]) base[to_sh[i + j]] = v[j];
      }
    }
    // a bad step of the path ends the entry's move: the rows behind it stay
    if (__syncthreads_or(end)) break;
  }
}

// ---------------------------------------------------------------------------
// Pages: slab by slab, page dst[i] takes what page src[i] holds.
// ---------------------------------------------------------------------------
// The numbers travel in the launch: 480 pairs, or 16, which spare a small call the copy of 4 KB of parameters.
constexpr int COPY_THREADS = 256, COPY_AHEAD = 8, COPY_MANY = 480, COPY_FEW = 16;
template <int PAIRS>
struct Pairs {
  int src[PAIRS], dst[PAIRS];
};

// block: COPY_THREADS * each pieces of a page; x runs over a page's chunks, y over pairs and slabs
template <typename V, int PAIRS>
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(V* __restrict__ pool, const __grid_constant__ Pairs<PAIRS> pairs, int n,
                                                                  long long slab_pages, long long page_pieces, int chunks) {
  pdl_wait();
  pdl_trigger();
  const int chunk = blockIdx.x % chunks;
  const long long rest = blockIdx.x / chunks;
  const int pair = (int)(rest % n);
  const long long slab = rest / n;
  const V* from = pool + (slab * slab_pages + pairs.src[pair]) * page_pieces;
  V* to = pool + (slab * slab_pages + pairs.dst[pair]) * page_pieces;
  const long long step = (long long)chunks * COPY_THREADS;
  for (long long i = (long long)chunk * COPY_THREADS + threadIdx.x; i < page_pieces; i += step * COPY_AHEAD) {
    V v[COPY_AHEAD];
#pragma unroll
    for (int j = 0; j < COPY_AHEAD; ++j)
      if (i + j * step < page_pieces) v[j] = from[i + j * step];
#pragma unroll
    for (int j = 0; j < COPY_AHEAD; ++j)
      if (i + j * step < page_pieces) to[i + j * step] = v[j];
  }
}

// bytes of the widest access that every row starts and ends on: two at least, for the entries refuse odd addresses and odd sizes
static int piece_bytes(const void* p, long long row_bytes) {
  int b = 16;
  while (b > 2 && ((uintptr_t)p % b || row_bytes % b)) b >>= 1;
  return b;
}
template <typename F>
static int with_pieces(int bytes, F f) {
  switch (bytes) {
    case 16: return f(uint4{});
    case 8: return f(uint2{});
    case 4: return f((uint32_t)0);
    default: return f((uint16_t)0);
  }
}

template <int PAIRS>
static int copy_in(void* pool, long long slabs, long long num_pages, long long page_bytes, const long long* src, const long long* dst, int n,
                   int sms, cudaStream_t stream) {
  const int bytes = piece_bytes(pool, page_bytes);
  const long long pieces = page_bytes / bytes;
  for (int i0 = 0; i0 < n; i0 += PAIRS) {
    Pairs<PAIRS> p;
    const int here = std::min(PAIRS, n - i0);
    for (int i = 0; i < here; ++i) p.src[i] = (int)src[i0 + i], p.dst[i] = (int)dst[i0 + i];
    // a thread's eight pieces in flight, unless that leaves SMs without a block
    long long chunks = (pieces + COPY_THREADS * COPY_AHEAD - 1) / (COPY_THREADS * COPY_AHEAD);
    const long long most = (pieces + COPY_THREADS - 1) / COPY_THREADS;
    while (chunks < most && chunks * here * slabs < 4ll * sms) chunks = std::min(most, 2 * chunks);
    const long long blocks = chunks * here * slabs;
    if (blocks > 0x7fffffff) return refuse(ST_BAD_SIZE, "copy_pages: %lld blocks", blocks);
    const int status = with_pieces(bytes, [&](auto v) {
      using V = decltype(v);
      launch_pdl(copy_pages_kernel<V, PAIRS>, dim3((unsigned)blocks), dim3(COPY_THREADS), 0, stream, (V*)pool, p, here, num_pages, pieces,
                 (int)chunks);
      return launched();
    });
    if (status != ST_OK) return status;
  }
  return ST_OK;
}

}  // namespace drafts
}  // namespace srlm

using namespace srlm;
using namespace srlm::drafts;

// parents [T]: of every token, its parent's place among its entry's tokens, or -1.  mask [T, words].
extern "C" int srlm_draft_tree(const int* parents, const int* cu_q, const int* kv_lens, int* positions, int* mask, int words, int n, int T,
                               int window, int* err, cudaStream_t stream) {
  if (n <= 0 || T <= 0) return ST_OK;
  if (words <= 0 || words > 65535 || window < 0 || !err) return refuse(ST_BAD_SIZE, "draft_tree: words=%d window=%d", words, window);
  const int most = std::min(T, 32 * words);
  launch_pdl(draft_tree_kernel, dim3(n, std::min(65535, (most + TREE_THREADS - 1) / TREE_THREADS)), dim3(TREE_THREADS), 0, stream, parents,
             cu_q, kv_lens, positions, mask, words, T, window, err);
  return launched();
}

// path [n, cap], count [n], next [n].
extern "C" int srlm_accept_drafts(const int* tokens, const int* parents, const int* targets, const int* cu_q, int n, int T, int* path,
                                  int cap, int* count, int* next, int* err, cudaStream_t stream) {
  if (n <= 0) return ST_OK;
  if (cap <= 0 || !err) return refuse(ST_BAD_SIZE, "accept_drafts: room for %d tokens of a path", cap);
  launch_pdl(accept_drafts_kernel, dim3(n), dim3(32), 0, stream, tokens, parents, targets, cu_q, T, path, cap, count, next, err);
  return launched();
}

// pool [slabs, num_pages, nkv, page_size, row_bytes].
extern "C" int srlm_keep_drafts(void* pool, long long slabs, long long num_pages, int nkv, int page_size, long long row_bytes,
                                const int* block_table, int table_stride, const int* cu_q, const int* kv_lens, const int* path, int cap,
                                const int* count, int n, int* err, cudaStream_t stream) {
  if (n <= 0) return ST_OK;
  if (slabs <= 0 || num_pages <= 0 || nkv <= 0 || page_size <= 0 || row_bytes <= 0 || row_bytes % 2 || table_stride <= 0 || cap <= 0 ||
      n > 65535 || slabs > (1 << 20) || num_pages > 0x7fffffff || row_bytes > (1 << 20) || nkv > (1 << 20) || !err)
    return refuse(ST_BAD_SIZE, "keep_drafts: slabs=%lld pages=%lld nkv=%d page_size=%d row=%lld bytes entries=%d", slabs, num_pages, nkv,
                  page_size, row_bytes, n);
  if ((uintptr_t)pool % 2) return refuse(ST_BAD_ALIGN, "keep_drafts: the pool starts on an odd address");
  const int bytes = piece_bytes(pool, row_bytes);
  const long long pieces = row_bytes / bytes, columns = slabs * nkv * pieces, blocks = (columns + KEEP_THREADS - 1) / KEEP_THREADS;
  if (blocks > 0x7fffffff) return refuse(ST_BAD_SIZE, "keep_drafts: %lld columns", columns);
  return with_pieces(bytes, [&](auto v) {
    using V = decltype(v);
    launch_pdl(keep_drafts_kernel<V>, dim3((unsigned)blocks, n), dim3(KEEP_THREADS), 0, stream, (V*)pool, block_table, table_stride, cu_q,
               kv_lens, path, cap, count, (int)slabs, (int)num_pages, nkv, page_size, (int)pieces, err);
    return launched();
  });
}

// Kernels that a copy of n pages launches.
extern "C" int srlm_copy_pages_launches(int n) { return n <= 0 ? 0 : n <= COPY_FEW ? 1 : (n + COPY_MANY - 1) / COPY_MANY; }

// pool [slabs, num_pages, page_bytes]; src, dst: host arrays of n page numbers.  No page is written twice, none is both read
// and written.
extern "C" int srlm_copy_pages(void* pool, long long slabs, long long num_pages, long long page_bytes, const long long* src,
                               const long long* dst, int n, int sms, cudaStream_t stream) {
  if (n <= 0) return ST_OK;
  if (slabs <= 0 || num_pages <= 0 || num_pages > 0x7fffffff || page_bytes <= 0 || page_bytes % 2 || slabs > (1 << 20) || sms <= 0)
    return refuse(ST_BAD_SIZE, "copy_pages: slabs=%lld pages=%lld of %lld bytes", slabs, num_pages, page_bytes);
  if ((uintptr_t)pool % 2) return refuse(ST_BAD_ALIGN, "copy_pages: the pool starts on an odd address");
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
      return refuse(ST_BAD_SIZE, "copy_pages: page %lld or %lld is outside the pool of %lld", src[i], dst[i], num_pages);
  try {
    std::vector<long long> to(dst, dst + n);
    std::sort(to.begin(), to.end());
    for (int i = 0; i < n; ++i) {
      if (i && to[i] == to[i - 1]) return refuse(ST_BAD_SIZE, "copy_pages: page %lld would be written twice", to[i]);
      if (std::binary_search(to.begin(), to.end(), src[i]))
        return refuse(ST_BAD_SIZE, "copy_pages: page %lld is both read and written", src[i]);
    }
  } catch (...) {
    return refuse(ST_BAD_SIZE, "copy_pages: no host memory for %d page numbers", n);
  }
  return n <= COPY_FEW ? copy_in<COPY_FEW>(pool, slabs, num_pages, page_bytes, src, dst, n, sms, stream)
                       : copy_in<COPY_MANY>(pool, slabs, num_pages, page_bytes, src, dst, n, sms, stream);
}
