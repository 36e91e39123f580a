// Attention for drafted tokens on bfloat16 tensor cores at warp level (mma.sync m16n8k16, float32 accumulation): heads of any
// multiple of 16 up to 256, any page size.  What a row sees and how the work is divided:
// tree_attention.cuh.
//
// A block's four warps share a tile of 64 keys, fetched with cp.async through the block table (the rows' addresses are found
// a tile ahead, so that a fetch is one shared-memory read and a copy).  Warps are KEY_WARPS ways along the keys and 4 / KEY_WARPS
// ways along the rows, 16 rows each: a chain of a few tokens (one group of 16 rows) has every warp at a quarter of the keys, a
// tree its own rows.  The warps of a row add their shares through shared memory at the end of a piece.  A weight is rounded to
// bfloat16 for the product with the values, and it is the rounded one that enters the row's sum: the weights that the product sees add
// up to one.
//
// The products multiply a masked key's value by an exact zero, which is none for an infinity.  In tiles where rows see
// different keys (the drafted tokens, a window's edge) such values are taken out of the tile, and the rows that do see them
// get them back as they are written.
#include "mma_sync.cuh"
#include "tree_attention.cuh"

namespace srlm {
namespace tree {

constexpr int M_KEYS = 64, M_THREADS = 128;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int HD_MAX, int KEY_WARPS, int STAGES>
struct MmaForm {
  static constexpr int ROW_WARPS = 4 / KEY_WARPS, ROWS = 16 * ROW_WARPS;
  static size_t smem(int hd) {
    const size_t ld = (hd + 8) * sizeof(bf16);
    const size_t tiles = STAGES * 2 * M_KEYS * ld, join = KEY_WARPS > 1 ? sizeof(float) * 4 * 16 * (hd + 2) : 0;
    return ROWS * ld + (tiles > join ? tiles : join);
  }
};

// Blocks on an SM, by registers and shared memory: the grid is what runs at once.
__host__ __device__ constexpr int mma_blocks(int hd) { return hd <= 64 ? 3 : hd <= 128 ? 2 : 1; }

template <int HD_MAX, int KEY_WARPS, int STAGES>
__global__ void __launch_bounds__(M_THREADS, mma_blocks(HD_MAX)) tree_mma_kernel(const __grid_constant__ Args a) {
  using Form = MmaForm<HD_MAX, KEY_WARPS, STAGES>;
  constexpr int ROWS = Form::ROWS, WK = M_KEYS / KEY_WARPS;      // keys of a warp in a tile
  constexpr int KS = HD_MAX / 16, NO = HD_MAX / 8, NS = WK / 8;
  extern __shared__ __align__(16) uint8_t tree_smem[];
  __shared__ long long at_sh[STAGES + 1][M_KEYS];                // first element of a key's row; -1: no key of the entry
  __shared__ int loose_sh;
  const int hd = a.hd, ld = hd + 8, chunks = hd >> 3;
  bf16* q_sh = reinterpret_cast<bf16*>(tree_smem);               // [ROWS][ld]
  bf16* kv_sh = q_sh + ROWS * ld;                                // [STAGES][keys | values][64][ld]
  const int tile_elems = M_KEYS * ld;
  const bf16* q = (const bf16*)a.q;
  const bf16* kc = (const bf16*)a.k_cache;
  const bf16* vc = (const bf16*)a.v_cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, mi = lane >> 3;
  const int row_warp = warp / KEY_WARPS, key0 = (warp % KEY_WARPS) * WK;
  const int g = a.g;
  pdl_wait();
  pdl_trigger();
  Walk<ROWS, M_KEYS> walk;
  walk.init(a, blockIdx.x == 0);
  Piece w;
  if (threadIdx.x == 0) leave_no_unit(a);
  while (walk.next(a, w)) {
    if (threadIdx.x == 0) leave_unit(a, walk, w);
    const Entry& x = w.x;
    const int r0 = w.block * ROWS, rows = min(ROWS, x.q_len * g - r0), tiles = w.tile_hi - w.tile_lo;
    const int* table = a.block_table + (size_t)w.e * a.table_stride;
    const int first_key = a.window > 0 ? max(0, x.start - a.window + 1) : 0;
    auto locate = [&](int t) {                                   // places of the piece's tile t
      if (tid < M_KEYS) {
        const int j = (w.tile_lo + t) * M_KEYS + tid;
        at_sh[t % (STAGES + 1)][tid] = t < tiles && j >= first_key && j < x.kv_len ? row_of_key(a, table, j, w.kvh) * hd : -1;
      }
    };
    auto fetch = [&](int t) {
      if (t < tiles) {
        bf16* kd = kv_sh + (t % STAGES) * 2 * tile_elems;
        bf16* vd = kd + tile_elems;
        const long long* at = at_sh[t % (STAGES + 1)];
        for (int i = tid; i < M_KEYS * chunks; i += M_THREADS) {
          const int key = i / chunks, c = (i - key * chunks) * 8;
          const long long row = at[key];
          cp_async_16(kd + key * ld + c, kc + (row < 0 ? 0 : row + c), row >= 0);
          cp_async_16(vd + key * ld + c, vc + (row < 0 ? 0 : row + c), row >= 0);
        }
      }
      cp_async_commit();
    };
    for (int t = 0; t < STAGES; ++t) locate(t);
    if (tid == 0) loose_sh = 0;
    for (int i = tid; i < ROWS * chunks; i += M_THREADS) {
      const int row = i / chunks, c = (i - row * chunks) * 8, r = r0 + row;
      const bool there = row < rows;
      cp_async_16(q_sh + row * ld + c, there ? q + ((size_t)(x.q0 + r / g) * a.nq + w.kvh * g + r % g) * hd + c : q, there);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) fetch(t);

    uint32_t qf[KS][4];
    float o[NO][4], m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NO; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    // this thread's two rows, and the row's tokens
    const int ra = row_warp * 16 + (lane >> 2);
    int token[2], lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      token[i] = x.q0 + min(r0 + ra + 8 * i, x.q_len * g - 1) / g;
      lo[i] = first_key_of(a, token[i], x.start, x.kv_len);
    }
    const bool live = row_warp * 16 < rows;

    for (int t = 0; t < tiles; ++t) {
      cp_async_wait<STAGES - 2>();
      __syncthreads();                                           // tile t is there; tile t - 1 and its places are done with
      fetch(t + STAGES - 1);
      locate(t + STAGES);
      const int j0 = (w.tile_lo + t) * M_KEYS;
      const bool plain = j0 + M_KEYS <= x.start && (a.window <= 0 || j0 >= x.kv_len - a.window);
      Sight<(WK + 31) / 32> sight[2];
      if (!plain && live) {
        sight[0].words(a, token[0], j0 + key0, x.start);
        sight[1].words(a, token[1], j0 + key0, x.start);
      }
      bf16* kt = kv_sh + (t % STAGES) * 2 * tile_elems;
      bf16* vt = kt + tile_elems;
      if (!plain) {
        bool loose = false;
        for (int i = tid; i < M_KEYS * chunks; i += M_THREADS) {
          uint4* p = reinterpret_cast<uint4*>(vt + i / chunks * ld + i % chunks * 8);
          uint4 v = *p;
          const bool here = take_loose(v);
          if (here) {
            *p = v;
            loose = true;
          }
        }
        if (loose) loose_sh = 1;
        __syncthreads();
      }
      if (t == 0)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          if (ks * 16 < hd) ldmatrix_x4(qf[ks], q_sh + (row_warp * 16 + (mi & 1) * 8 + (lane & 7)) * ld + (ks * 2 + (mi >> 1)) * 8);
      if (!live) continue;
      float s[NS][4];
#pragma unroll
      for (int nt = 0; nt < NS; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks * 16 < hd) {
#pragma unroll
          for (int nt = 0; nt < NS; nt += 2) {
            uint32_t b[4];
            ldmatrix_x4(b, kt + (key0 + (nt + (mi >> 1)) * 8 + (lane & 7)) * ld + (ks * 2 + (mi & 1)) * 8);
            mma_bf16(s[nt], qf[ks], b[0], b[1]);
            mma_bf16(s[nt + 1], qf[ks], b[2], b[3]);
          }
        }
      }
      if (!plain) {
        constexpr int NW = (WK + 31) / 32;
        uint32_t bits[2][NW];
#pragma unroll
        for (int i = 0; i < 2; ++i) sight[i].bits(bits[i], j0 + key0, x.start, x.kv_len, lo[i]);
#pragma unroll
        for (int nt = 0; nt < NS; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = nt * 8 + (lane & 3) * 2 + (i & 1);
            if (!((bits[i >> 1][(nt * 8) / 32] >> (k & 31)) & 1)) s[nt][i] = -CUDART_INF_F;      // (the score scale is positive)
          }
      }
      float mx[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
      for (int nt = 0; nt < NS; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i >> 1] = fmaxf(mx[i >> 1], s[nt][i]);
      float base[2], sum[2] = {0.f, 0.f}, alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        mx[i] = fmaxf(mx[i] * a.scale_log2, m[i]);
        base[i] = mx[i] == -CUDART_INF_F ? 0.f : mx[i];
        alpha[i] = ex2(m[i] - base[i]);
        m[i] = mx[i];
      }
      uint32_t pf[NS / 2][4];
#pragma unroll
      for (int nt = 0; nt < NS; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t p = pack_bf16(ex2(fmaf(s[nt][2 * i], a.scale_log2, -base[i])), ex2(fmaf(s[nt][2 * i + 1], a.scale_log2, -base[i])));
          sum[i] += __uint_as_float(p << 16) + __uint_as_float(p & 0xffff0000u);
          pf[nt >> 1][(nt & 1) * 2 + i] = p;
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) l[i] = l[i] * alpha[i] + sum[i];     // (of this lane's keys; the lanes add up at the end)
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int dn = 0; dn < NO; ++dn) {
          o[dn][0] *= alpha[0];
          o[dn][1] *= alpha[0];
          o[dn][2] *= alpha[1];
          o[dn][3] *= alpha[1];
        }
      }
#pragma unroll
      for (int kk = 0; kk < NS / 2; ++kk) {
#pragma unroll
        for (int dn = 0; dn < NO; dn += 2) {
          if (dn * 8 < hd) {
            uint32_t b[4];
            ldmatrix_x4_trans(b, vt + (key0 + kk * 16 + (mi & 1) * 8 + (lane & 7)) * ld + (dn + (mi >> 1)) * 8);
            mma_bf16(o[dn], pf[kk], b[0], b[1]);
            mma_bf16(o[dn + 1], pf[kk], b[2], b[3]);
          }
        }
      }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    __syncthreads();                                             // the tiles' memory is free
    const bool loose = loose_sh != 0, whole = w.begins && w.ends;
    const size_t slab = slab_of(blockIdx.x, w.begins);
    auto out_of = [&](int row) {
      const int r = r0 + row;
      return (bf16*)a.out + ((size_t)(x.q0 + r / g) * a.nq + w.kvh * g + r % g) * hd;
    };
    // two neighbouring numbers of a row
    auto put = [&](int row, bf16* dst, int d, float v0, float v1, float inv) {
      if (whole) {
        *reinterpret_cast<uint32_t*>(dst + d) = pack_bf16(v0 * inv, v1 * inv);
      } else {
        float* part = a.part_o + (slab * hd + d) * ROWS + row;
        part[0] = v0;
        part[ROWS] = v1;
      }
    };
    if constexpr (KEY_WARPS == 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = ra + 8 * i;
        if (row >= rows) continue;
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        bf16* dst = out_of(row);
        if (!whole && (lane & 3) == 0) *reinterpret_cast<float2*>(a.part_ml + (slab * ROWS + row) * 2) = make_float2(m[i], l[i]);
#pragma unroll
        for (int dn = 0; dn < NO; ++dn)
          if (dn * 8 < hd) put(row, dst, dn * 8 + (lane & 3) * 2, o[dn][2 * i], o[dn][2 * i + 1], inv);
      }
    } else {
      float* o_sh = reinterpret_cast<float*>(kv_sh);             // [4 warps][16][hd]
      float2* ml_sh = reinterpret_cast<float2*>(o_sh + 4 * 16 * hd);   // [4 warps][16]
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = (lane >> 2) + 8 * i;
        if ((lane & 3) == 0) ml_sh[warp * 16 + row] = make_float2(m[i], l[i]);
#pragma unroll
        for (int dn = 0; dn < NO; ++dn)
          if (dn * 8 < hd)
            *reinterpret_cast<float2*>(o_sh + (warp * 16 + row) * hd + dn * 8 + (lane & 3) * 2) = make_float2(o[dn][2 * i], o[dn][2 * i + 1]);
      }
      __syncthreads();
      const int pairs = hd >> 1;
      for (int i = tid; i < ROWS * pairs; i += M_THREADS) {
        const int row = whole ? i / pairs : i % ROWS, d = (whole ? i - row * pairs : i / ROWS) * 2;      // (as they are stored side by side)
        if (row >= rows) continue;
        const int first = (row >> 4) * KEY_WARPS * 16 + (row & 15);      // the row in its first warp's share
        float M = -CUDART_INF_F, L = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
        for (int k = 0; k < KEY_WARPS; ++k) M = fmaxf(M, ml_sh[first + 16 * k].x);
        const float mb = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
        for (int k = 0; k < KEY_WARPS; ++k) {
          const float2 ml = ml_sh[first + 16 * k];
          const float f = ex2(ml.x - mb);
          const float2 v = *reinterpret_cast<const float2*>(o_sh + (first + 16 * k) * hd + d);
          L += f * ml.y;
          v0 += f * v.x;
          v1 += f * v.y;
        }
        if (!whole && d == 0) *reinterpret_cast<float2*>(a.part_ml + (slab * ROWS + row) * 2) = make_float2(M, L);
        put(row, out_of(row), d, v0, v1, L == 0.f ? 0.f : 1.f / L);
      }
    }
    __syncthreads();                                             // before the next piece's rows and tiles
    if (loose) {                                                 // (what a row sees of them, on top of the rest: that may hold some too)
      for (int i = tid; i < rows * hd; i += M_THREADS) {
        const int row = i / hd, d = i - row * hd;
        const float v = loose_values<bf16, M_KEYS>(a, x.start, x.kv_len, table, w.kvh, x.q0 + (r0 + row) / g, d, w.tile_lo, w.tile_hi);
        if (isfinite(v)) continue;
        if (whole) out_of(row)[d] = from_float<bf16>(to_float(out_of(row)[d]) + v);
        else a.part_o[(slab * hd + d) * ROWS + row] += v;
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// Warps along the keys: by the rows that an entry has at most (8 KV heads of 128, pages of 20, 8 entries behind 8,000 keys, us, four |
// two | one: 16 rows 60.7 | 63.0 | 68.9, 32 rows 104 | 65.5 | 77.6, 64 rows 183 | 114 | 83.2).
static int key_warps(int max_rows) { return max_rows <= 16 ? 4 : max_rows <= 32 ? 2 : 1; }

bool mma_takes(int hd) { return hd % 16 == 0 && hd <= 256; }
Form mma_form(int hd, int max_rows, int sms) { return Form{mma_blocks(hd) * sms, 64 / key_warps(max_rows), M_KEYS}; }

template <int HD_MAX, int KEY_WARPS, int STAGES>
static int run_form(const Args& a, int blocks, cudaStream_t stream) {
  using F = MmaForm<HD_MAX, KEY_WARPS, STAGES>;
  const int smem = (int)F::smem(a.hd), most = (int)F::smem(HD_MAX);
  static std::atomic<bool> have[64];
  const cudaError_t e = allow_smem((const void*)tree_mma_kernel<HD_MAX, KEY_WARPS, STAGES>, most, have);
  if (e != cudaSuccess) return refuse((int)e, "tree_attention: cannot get %d bytes of shared memory", most);
  launch_pdl(tree_mma_kernel<HD_MAX, KEY_WARPS, STAGES>, dim3(blocks), dim3(M_THREADS), smem, stream, a);
  launch_merge<bf16, F::ROWS, M_KEYS>(a, blocks, stream);
  return launched();
}
// Stages: as many as leave room for another block on the SM.
template <int HD_MAX, int STAGES, int STAGES_ROWS>
static int run_rows(const Args& a, int max_rows, int sms, cudaStream_t stream) {
  const int blocks = mma_form(a.hd, max_rows, sms).blocks;
  switch (key_warps(max_rows)) {
    case 4: return run_form<HD_MAX, 4, STAGES>(a, blocks, stream);
    case 2: return run_form<HD_MAX, 2, STAGES>(a, blocks, stream);
    default: return run_form<HD_MAX, 1, STAGES_ROWS>(a, blocks, stream);
  }
}
int run_mma(const Args& a, int max_rows, int sms, cudaStream_t stream) {
  if (a.hd <= 64) return run_rows<64, 3, 3>(a, max_rows, sms, stream);
  if (a.hd <= 128) return run_rows<128, 3, 2>(a, max_rows, sms, stream);
  return run_rows<256, 2, 2>(a, max_rows, sms, stream);
}

}  // namespace tree
}  // namespace srlm
