// Attention for drafted tokens on the 5th-generation tensor cores: bfloat16 heads of 64 or 128, pages that a TMA box
// covers.  What a row sees and how the work is divided: tree_attention.cuh.
//
// A unit is up to 128 rows (token x query head of a KV group), the M of one MMA, over tiles of 128 keys:
//     S = Q . K^T      both in shared memory, K-major
//     O += P . V       P in tensor memory (bfloat16, over the columns of S), V in shared memory, MN-major
// Trees have few rows, so it is the keys that keep the tensor core busy: the piece's tiles go to two streams in turn, each
// with an S and an O of its own in tensor memory (512 columns in all) and four softmax warps, a thread a row.  While one stream's
// warps form the weights of a tile, the tensor core works for the other, and three stages of keys and values (six of heads of
// 64) are in flight.  At the end of a piece the two streams' sums are joined as they are read from tensor memory (a warp reads
// the same lanes of both; each stream's warps write half of the columns).
// Warps 0, 10 and 11 fetch tiles of keys and of values in turn (a lane a page box; an issue takes 70 ns beside busy softmax warps, and a
// tile of pages of 16 has 16 boxes), one thread of warp 1 issues the MMAs, warps 2-5 and 6-9 are the streams' softmax.  The softmax
// bounds calls of many rows: 1.45 us a tile and stream, of which 0.55 are its exponentials alone, beside 0.9 us of products.  A block
// stays for all of its pieces: the fetches run ahead across them, and the block count is the SMs'.
//
// A weight is rounded to bfloat16 for the product with the values, which is what the MMA takes; a row's sum is of the weights before that
// rounding, each at most 2^-8 of itself from what the product sees.  Outputs are 0.0023 of their size off 64 bits, 0.0017 of it from their
// own type (the warp-level form, whose sum is of the rounded weights: 0.0021); unpacking the rounded pairs for the sum would be two more
// instructions a pair in the softmax, which bounds calls of many rows.
// O is rescaled only when a row's maximum has grown by more than 2^8: until then the old one stays the reference of the exponentials, and
// the division by the sum makes it exact.
// Every wait is bounded; one that runs out raises the error word and ends the block's work.
#include "attention_tcgen05.cuh"
#include "tree_attention.cuh"

namespace srlm {
namespace tree {

using namespace fmha;

constexpr int T_ROWS = 128, T_KEYS = 128, T_THREADS = 384, T_SOFTMAX = 256, T_PRODUCERS = 3;
constexpr float T_RESCALE_ABOVE = 8.f;             // log2 of the growth of a row's maximum that O is rescaled for

template <int HD>
struct TmaForm {
  static constexpr int TILE = T_KEYS * HD * 2;     // bytes of a tile of keys, values or rows
  static constexpr int STAGES = HD == 128 ? 3 : 6;
  static constexpr int SMEM = TILE * (1 + 2 * STAGES) + 1024 + (4 * STAGES + 9) * 8;
};

__device__ __forceinline__ bool elected() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// Scores of keys that the row does not see become -inf (the score scale is positive): a weight of zero.
__device__ __forceinline__ void mask_row(Row& r, const uint32_t (&bits)[4]) {
  auto part = [&](uint32_t (&v)[32], uint32_t b) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = (b >> j) & 1 ? v[j] : 0xff800000u;
  };
  part(r.a, bits[0]);
  part(r.b, bits[1]);
  part(r.c, bits[2]);
  part(r.d, bits[3]);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float row_top(const Row& r) {
  float m[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
  auto part = [&](const uint32_t (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) m[(j >> 1) & 3] = max3(m[(j >> 1) & 3], __uint_as_float(v[j]), __uint_as_float(v[j + 1]));
  };
  part(r.a);
  part(r.b);
  part(r.c);
  part(r.d);
  return max3(fmaxf(m[0], m[1]), m[2], m[3]);
}
// The weights exp2(S * scale - base) of 64 keys as bfloat16 pairs over columns of S; their sum, pairs by pairs.
__device__ __forceinline__ float2 half_exp(uint32_t addr, const uint32_t (&va)[32], const uint32_t (&vb)[32], float scale, float base) {
  const float2 sc = make_float2(scale, scale), nb = make_float2(-base, -base);
  float2 s0 = make_float2(0.f, 0.f), s1 = s0;
  auto part = [&](const uint32_t (&v)[32], uint32_t at) {
    uint32_t pk[16];
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      float2 x = fma2(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), sc, nb);
      float2 y = fma2(make_float2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])), sc, nb);
      x = make_float2(ex2(x.x), ex2(x.y));
      y = make_float2(ex2(y.x), ex2(y.y));
      pk[j >> 1] = pack2(x.x, x.y);
      pk[(j >> 1) + 1] = pack2(y.x, y.y);
      s0 = add2(s0, x);
      s1 = add2(s1, y);
    }
    tmem_st16(at, pk);
  };
  part(va, addr);
  part(vb, addr + 16);
  return add2(s0, s1);
}

template <int HD>
__global__ void __launch_bounds__(T_THREADS, 1)
tree_tcgen05_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a) {
  using Form = TmaForm<HD>;
  constexpr int TILE = Form::TILE, STAGES = Form::STAGES, CHUNKS = HD / 8;
  extern __shared__ uint8_t tree_smem_raw[];
  uint8_t* smem = tree_smem_raw + ((1024u - (s32(tree_smem_raw) & 1023u)) & 1023u);
  uint8_t* q_t = smem;
  uint8_t* k_t = q_t + TILE;                       // [STAGES]
  uint8_t* v_t = k_t + STAGES * TILE;              // [STAGES]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(v_t + STAGES * TILE);
  uint64_t* k_empty = k_full + STAGES;
  uint64_t* v_full = k_empty + STAGES;
  uint64_t* v_empty = v_full + STAGES;
  uint64_t* s_full = v_empty + STAGES;             // [2]: per stream
  uint64_t* p_ready = s_full + 2;                  // [2]
  uint64_t* p_half = p_ready + 2;                  // [2]: the weights of a tile's first 64 keys
  uint64_t* o_done = p_half + 2;                   // [2]
  uint64_t* q_full = o_done + 2;
  __shared__ Walk<T_ROWS, T_KEYS> walk_sh;
  __shared__ Piece piece_sh[2];
  __shared__ int more_sh;
  __shared__ uint32_t tmem_sh;
  __shared__ int loose_sh, failed_sh;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&p_half[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(q_full, T_SOFTMAX / 32);
    loose_sh = failed_sh = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&tmem_sh)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_sh;
  pdl_wait();
  pdl_trigger();

  const int g = a.g;
  using Walks = Walk<T_ROWS, T_KEYS>;
  Walks walk;
  if (warp <= 2 || warp >= 10) {
    walk.init(a, blockIdx.x == 0 && warp == 0);
    if (warp == 2 && lane == 0) walk_sh = walk;    // (the softmax warps keep theirs in shared memory: its numbers would cost them registers)
  }

  const int ps = a.page_size, box_rows = ps < T_KEYS ? ps : T_KEYS;
  if (warp == 0 || warp >= 10) {
    // ---------------- TMA producers ----------------
    const int producer = warp == 0 ? 0 : warp - 9, boxes = T_KEYS / box_rows;
    const int shift = 31 - __clz(ps);
    const bool pages = ps & (ps - 1);              // of no power of two
    int job = 0, k = 0;                            // tiles of keys and of values in turn, so far; tiles of keys
    bool ok = true;
    Piece w;
    while (ok && walk.next(a, w)) {
      const int* table = a.block_table + (size_t)w.e * a.table_stride;
      const int first = a.window > 0 ? max(0, w.x.start - a.window + 1) : 0;
      // the lane's page of a tile, looked up a tile ahead (behind the entry's last key: page 0, which nobody sees)
      auto page_of = [&](int t) {
        const int key = t * T_KEYS + lane * box_rows;
        return lane < boxes && t < w.tile_hi && key < w.x.kv_len ? table[pages ? key / ps : key >> shift] : 0;
      };
      int page_next = page_of(w.tile_lo);
      for (int t = w.tile_lo; t < w.tile_hi && ok; ++t, ++k) {
        const int s = k % STAGES;
        int page = page_next;
        page_next = page_of(t + 1);
        const int key = t * T_KEYS + lane * box_rows;
        if (page < 0 || page >= a.num_pages) {
          if (key + box_rows > first) atomicExch(a.err_flag, ERR_PAGE);      // (pages behind a window are given back)
          page = 0;
        }
        const int row = (page * a.nkv + w.kvh) * ps + (pages ? key % ps : key & (ps - 1));
        for (int values = 0; values < 2; ++values, ++job) {
          if (job % T_PRODUCERS != producer) continue;
          uint64_t *full = values ? &v_full[s] : &k_full[s], *empty = values ? &v_empty[s] : &k_empty[s];
          ok = __all_sync(0xffffffffu, mbar_wait(empty, ((k / STAGES) & 1) ^ 1, a.err_flag, 81));
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(full, TILE);
          __syncwarp();
          if (lane < boxes) {
            uint8_t* tile = (values ? v_t : k_t) + s * TILE + lane * box_rows * 128;
#pragma unroll
            for (int c = 0; c < HD; c += 64) tma_load_2d(tile + c * (T_KEYS * 2), values ? &map_v : &map_k, full, c, row);
          }
        }
      }
    }
    if (!ok)                                       // copies in flight end before the block does
      for (int back = 1; back <= STAGES && back <= k; ++back) {
        mbar_wait(&k_full[(k - back) % STAGES], ((k - back) / STAGES) & 1, a.err_flag, 82);
        mbar_wait(&v_full[(k - back) % STAGES], ((k - back) / STAGES) & 1, a.err_flag, 82);
      }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    // The whole warp goes through the same steps and one elected lane issues: the operands then are the warp's, and an issue costs no
    // moves between register files (a loop that one lane alone goes through: 144 cycles an MMA, where it takes 64).
    const uint32_t idesc_s = umma_idesc(T_KEYS, false), idesc_o = umma_idesc(HD, true);
    // descriptors: the start address sits in the low bits, in units of 16 bytes, so a k-step is an addition
    const uint64_t q_desc = umma_desc(s32(q_t), 0, 1024), k_desc = umma_desc(s32(k_t), 0, 1024);
    const uint64_t v_desc = umma_desc(s32(v_t), T_KEYS * 128, 1024);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const bool issues = elected();
    int s_k = 0, s_v = 0, piece = 0;               // ring stages of the next keys and values, pieces so far
    uint32_t k_phase = 0, v_phase = 0, p_phase = 0;        // the waits' parities, a bit a stream in the last
    bool ok = true;
    Piece w;
    if (lane == 0) leave_no_unit(a);
    while (walk.next(a, w)) {
      if (lane == 0) leave_unit(a, walk, w);
      const int tiles = __shfl_sync(0xffffffffu, w.tile_hi - w.tile_lo, 0);
      auto issue_s = [&](int i) {                  // S_i = Q . K^T of the next keys
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&k_full[s_k], k_phase, a.err_flag, 83));
        if (!ok) return;
        fence_after();
        const uint64_t kd = k_desc + (uint64_t)(s_k * (TILE >> 4));
        if (issues) {
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * (T_KEYS * 128) + (ks & 3) * 32) >> 4;      // panel, then 32 bytes a k-step
            umma_bf16(tm + i * 128, q_desc + off, kd + off, idesc_s, ks != 0);
          }
          umma_commit(&s_full[i]);
          umma_commit(&k_empty[s_k]);
        }
        __syncwarp();
        if (++s_k == STAGES) s_k = 0, k_phase ^= 1;
      };
      ok = ok && __all_sync(0xffffffffu, mbar_wait(q_full, piece & 1, a.err_flag, 84));
      ++piece;
      if (!ok) break;
      fence_after();
      issue_s(0);
      if (tiles > 1) issue_s(1);
      for (int t = 0; t < tiles && ok; ++t) {
        const int i = t & 1;
        const uint64_t vd = v_desc + (uint64_t)(s_v * (TILE >> 4));
        const uint32_t d = tm + 256 + i * 128, p = tm + i * 128;
        ok = __all_sync(0xffffffffu, mbar_wait(&v_full[s_v], v_phase, a.err_flag, 85) &&
                                         mbar_wait(&p_half[i], (p_phase >> i) & 1, a.err_flag, 86));
        if (!ok) break;
        fence_after();
        if (issues) {
#pragma unroll
          for (int kk = 0; kk < T_KEYS / 32; ++kk)   // 16 keys: 8 columns of pairs, 2048 bytes of values
            umma_bf16_ts(d, p + kk * 8, vd + kk * (2048 >> 4), idesc_o, t > 1 || kk > 0);
        }
        __syncwarp();
        ok = __all_sync(0xffffffffu, mbar_wait(&p_ready[i], (p_phase >> i) & 1, a.err_flag, 91));
        if (!ok) break;
        p_phase ^= 1u << i;
        fence_after();
        if (issues) {
#pragma unroll
          for (int kk = T_KEYS / 32; kk < T_KEYS / 16; ++kk) umma_bf16_ts(d, p + kk * 8, vd + kk * (2048 >> 4), idesc_o, 1);
          umma_commit(&o_done[i]);
          umma_commit(&v_empty[s_v]);
        }
        __syncwarp();
        if (++s_v == STAGES) s_v = 0, v_phase ^= 1;
        if (t + 2 < tiles) issue_s(i);
      }
      if (!ok) break;
    }
  } else {
    // ---------------- softmax: a thread a row ----------------
    const int i = (warp - 2) >> 2, ew = warp & 3, row = ew * 32 + lane, st = threadIdx.x - 64;
    const uint32_t lane_addr = (uint32_t)(ew * 32) << 16;
    const uint32_t s_addr = tmem + i * 128 + lane_addr, o_addr = tmem + 256 + i * 128 + lane_addr;
    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(T_SOFTMAX) : "memory"); };      // both streams
    uint32_t done = 0;                             // tiles of this stream so far
    int k = 0;                                     // tiles of the block so far
    bool ok = true;
    if (threadIdx.x == 64) more_sh = walk_sh.next(a, piece_sh[0]);
    meet();
    for (int n = 0; more_sh; n ^= 1) {
      const Piece& w = piece_sh[n];
      const Entry& x = w.x;
      const int rows_total = x.q_len * g, r0 = w.block * T_ROWS, rows = min(T_ROWS, rows_total - r0), tiles = w.tile_hi - w.tile_lo;
      const int first = a.window > 0 ? max(0, x.start - a.window + 1) : 0;
      // the rows -> shared memory, swizzled (zeros behind the last), eight loads of a thread in flight; the products that read the last
      // piece's are done (their tiles were waited for)
      const bf16* q = (const bf16*)a.q;
      constexpr int QB = 8;
#pragma unroll 1
      for (int base = st; base < T_ROWS * CHUNKS; base += T_SOFTMAX * QB) {
        uint4 v[QB];
#pragma unroll
        for (int j = 0; j < QB; ++j) {
          const int idx = base + j * T_SOFTMAX, rr = idx / CHUNKS, c = idx % CHUNKS, r = r0 + rr;
          v[j] = make_uint4(0, 0, 0, 0);
          if (rr < rows) v[j] = __ldg(reinterpret_cast<const uint4*>(q + ((size_t)(x.q0 + r / g) * a.nq + w.kvh * g + r % g) * HD + c * 8));
        }
#pragma unroll
        for (int j = 0; j < QB; ++j) {
          const int idx = base + j * T_SOFTMAX, rr = idx / CHUNKS, c = idx % CHUNKS;
          if (rr < T_ROWS)
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(tile_addr(s32(q_t), rr, c)), "r"(v[j].x), "r"(v[j].y), "r"(v[j].z),
                         "r"(v[j].w) : "memory");
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);

      const int r = min(r0 + row, rows_total - 1), token = x.q0 + r / g;
      const bool live = ew * 32 < rows;            // some row of the warp is one
      float m_run = -CUDART_INF_F, l_run = 0.f;
      bool any = false;
      for (int t = i; t < tiles && ok; t += 2, ++done, any = true) {
        const int j0 = (w.tile_lo + t) * T_KEYS;
        // every row sees every key of a tile between the window's last edge and the drafted tokens
        const bool plain = j0 + T_KEYS <= x.start && (a.window <= 0 || j0 >= x.kv_len - a.window);
        uint32_t bits[4];
        if (!plain && live) {
          Sight<4> sight;
          sight.words(a, token, j0, x.start);
          sight.bits(bits, j0, x.start, x.kv_len, first_key_of(a, token, x.start, x.kv_len));
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[i], done & 1, a.err_flag, 87));
        if (!ok) break;
        fence_after();
        if (!plain) {
          // values of no key of the entry become zeros, and those that are no numbers are taken out
          const int s = (k + t) % STAGES;
          ok = __all_sync(0xffffffffu, mbar_wait(&v_full[s], ((k + t) / STAGES) & 1, a.err_flag, 88));
          if (!ok) break;
          uint8_t* vt = v_t + s * TILE;
          const int behind = x.kv_len - j0, edge = a.window > 0 ? x.kv_len - a.window - j0 : 0;      // some row does not see keys in front of the edge
          const int from = edge > 0 ? 0 : max(x.start - j0, 0);
          bool loose = false;
#pragma unroll 1
          for (int idx = from * CHUNKS + row; idx < T_KEYS * CHUNKS; idx += 128) {
            const int key = idx / CHUNKS;
            uint4* at = reinterpret_cast<uint4*>(vt + tile_addr(0, key, idx % CHUNKS));
            uint4 v = make_uint4(0, 0, 0, 0);
            bool change = true;
            if (key < behind && j0 + key >= first) {
              v = *at;
              loose |= change = take_loose(v);
            }
            if (change) *at = v;
          }
          if (loose) loose_sh = 1;
          fence_async_smem();
          __syncwarp();                            // a warp of no rows arrives for all its lanes at once: each has written and fenced by then
        }
        if (live) {
          Row srow;
          load_row(s_addr, srow);
          if (!plain) mask_row(srow, bits);
          const float mx = row_top(srow) * a.scale_log2;
          const bool grow = mx > m_run + T_RESCALE_ABOVE || m_run == -CUDART_INF_F;
          const float m_new = grow ? fmaxf(mx, m_run) : m_run;
          if (any && __any_sync(0xffffffffu, m_new != m_run)) {
            const float alpha = m_new == m_run ? 1.f : ex2(m_run - m_new);      // (from -inf: 0)
            ok = __all_sync(0xffffffffu, mbar_wait(&o_done[i], (done - 1) & 1, a.err_flag, 89));         // the tile before is in O
            fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              uint32_t v[16];
              tmem_ld16(o_addr + c, v);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
              tmem_st16(o_addr + c, v);
            }
            l_run *= alpha;
          }
          m_run = m_new;
          const float base = m_run == -CUDART_INF_F ? 0.f : m_run;
          const float2 s0 = half_exp(s_addr, srow.a, srow.b, a.scale_log2, base);
          tmem_wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_half[i]);
          const float2 s1 = add2(s0, half_exp(s_addr + 32, srow.c, srow.d, a.scale_log2, base));
          l_run += s1.x + s1.y;
          tmem_wait_st();
        } else if (lane == 0) {
          mbar_arrive(&p_half[i]);
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[i]);
      }
      if (ok && any) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[i], (done - 1) & 1, a.err_flag, 90));
      k += tiles;
      if (!ok) failed_sh = 1;
      if (ok && any && live) {                     // the row's reference and sum over the first columns of S, whose weights are used up
        uint32_t ml[16] = {__float_as_uint(m_run), __float_as_uint(l_run)};
        tmem_st16(s_addr, ml);
        tmem_wait_st();
      }
      Piece* following = &piece_sh[n ^ 1];
      const int more = threadIdx.x == 64 ? walk_sh.next(a, *following) : 0;      // (while the other stream ends)
      fence_before();
      meet();
      fence_after();
      ok = ok && !failed_sh;
      if (ok && live) {
        // both streams' sums of the row, half of the columns each
        const bool two = tiles > 1;
        uint32_t ml0[16], ml1[16];
        tmem_ld16(tmem + lane_addr, ml0);
        tmem_ld16(tmem + 128 + lane_addr, ml1);
        tmem_wait_ld();
        const float2 s0 = make_float2(__uint_as_float(ml0[0]), __uint_as_float(ml0[1]));
        const float2 s1 = make_float2(__uint_as_float(ml1[0]), __uint_as_float(ml1[1]));
        const float M = two ? fmaxf(s0.x, s1.x) : s0.x, mb = M == -CUDART_INF_F ? 0.f : M;
        const float f0 = ex2(s0.x - mb), f1 = two ? ex2(s1.x - mb) : 0.f;
        const float L = two ? f0 * s0.y + f1 * s1.y : f0 * s0.y;
        const bool mine = row < rows, whole = w.begins && w.ends;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const size_t slab = slab_of(blockIdx.x, w.begins);
        if (!whole && mine && i == 0) *reinterpret_cast<float2*>(a.part_ml + (slab * T_ROWS + row) * 2) = make_float2(M, L);
        bf16* dst = (bf16*)a.out + ((size_t)token * a.nq + w.kvh * g + r % g) * HD;
        const uint32_t both = tmem + 256 + lane_addr;
#pragma unroll 1
        for (int c = i * (HD / 2); c < (i + 1) * (HD / 2); c += 32) {
          uint32_t u[32], v[32];
          tmem_ld32(both + c, u);
          tmem_ld32(both + 128 + c, v);
          tmem_wait_ld();
          float o[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            o[j] = f0 * __uint_as_float(u[j]);
            if (two) o[j] = fmaf(f1, __uint_as_float(v[j]), o[j]);
          }
          if (mine && whole) {
#pragma unroll
            for (int n8 = 0; n8 < 32; n8 += 8)
              *reinterpret_cast<uint4*>(dst + c + n8) = make_uint4(pack2(o[n8] * inv, o[n8 + 1] * inv), pack2(o[n8 + 2] * inv, o[n8 + 3] * inv),
                                                                   pack2(o[n8 + 4] * inv, o[n8 + 5] * inv), pack2(o[n8 + 6] * inv, o[n8 + 7] * inv));
          } else if (mine) {
#pragma unroll
            for (int j = 0; j < 32; ++j) a.part_o[(slab * HD + c + j) * T_ROWS + row] = o[j];
          }
        }
        if (loose_sh && mine)                      // (what a row sees of them, on top of the rest: that may hold some too)
#pragma unroll 1
          for (int c = i * (HD / 2); c < (i + 1) * (HD / 2); ++c) {
            const float v = loose_values<bf16, T_KEYS>(a, x.start, x.kv_len, a.block_table + (size_t)w.e * a.table_stride, w.kvh, token,
                                                       c, w.tile_lo, w.tile_hi);
            if (!isfinite(v)) {
              if (whole) dst[c] = from_float<bf16>(to_float(dst[c]) + v);
              else a.part_o[(slab * HD + c) * T_ROWS + row] += v;
            }
          }
        fence_before();
      }
      if (threadIdx.x == 64) more_sh = more;
      meet();                                      // O, S and the rows are free
      if (st == 0) loose_sh = 0;                   // (read before the meeting, set behind the next piece's first tile)
      if (!ok) break;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---------------------------------------------------------------------------
static bool tensor_map(CUtensorMap* out, const void* ptr, long long rows, int hd, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)hd * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t elem[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool tcgen05_takes(int hd, int page_size) {
  return (hd == 64 || hd == 128) && (page_size == 8 || page_size == 16 || page_size == 32 || page_size == 64 ||
                                     (page_size > 0 && page_size % T_KEYS == 0));
}
Form tcgen05_form(int sms) { return Form{sms, T_ROWS, T_KEYS}; }

template <int HD>
static int run_form(const Args& a, int sms, cudaStream_t stream) {
  const int box_rows = min(a.page_size, T_KEYS);
  const long long rows = (long long)a.num_pages * a.nkv * a.page_size;
  CUtensorMap mk, mv;
  if (rows > 0x7fffffff || !tensor_map(&mk, a.k_cache, rows, HD, box_rows) || !tensor_map(&mv, a.v_cache, rows, HD, box_rows))
    return refuse(ST_BAD_SIZE, "tree_attention: the caches of %lld rows of %d cannot be mapped", rows, HD);
  static std::atomic<bool> have[64];
  const cudaError_t e = allow_smem((const void*)tree_tcgen05_kernel<HD>, TmaForm<HD>::SMEM, have);
  if (e != cudaSuccess) return refuse((int)e, "tree_attention: cannot get %d bytes of shared memory", TmaForm<HD>::SMEM);
  launch_pdl(tree_tcgen05_kernel<HD>, dim3(sms), dim3(T_THREADS), TmaForm<HD>::SMEM, stream, mk, mv, a);
  launch_merge<bf16, T_ROWS, T_KEYS>(a, sms, stream);
  return launched();
}
int run_tcgen05(const Args& a, int sms, cudaStream_t stream) {
  return a.hd == 64 ? run_form<64>(a, sms, stream) : run_form<128>(a, sms, stream);
}

}  // namespace tree
}  // namespace srlm
