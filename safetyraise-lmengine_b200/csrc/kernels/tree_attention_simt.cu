// Attention for drafted tokens in float32 arithmetic: the float32 path, and bfloat16 heads whose size the tensor-core forms
// do not take.  What a row sees and how the work is divided: tree_attention.cuh.
//
// A block walks its pieces' keys in tiles of 32.  A tile's keys and values are copied to shared memory once for all rows, the next
// tile in flight under the current one (float32 rows of whole 16-byte pieces asynchronously; others are read and converted), the
// places of the tile after it looked up meanwhile.  The four warps are KEY_WARPS ways along the tile's keys and 4 / KEY_WARPS ways
// along the rows, eight rows each: calls of few rows have every warp at a part of the keys.  For the scores the lanes of a warp are its
// keys times groups of its rows, so that a row's maximum and sum are reductions over lanes; for the outputs a lane holds the
// dimensions lane + 32 i, so that nothing but the weights passes through shared memory.  Bound by the latency of the FMAs' operands
// from shared memory (a 16-byte read feeds 32 of them at best), which more warps on the SM hide.
// A masked key's weight is an exact zero; values that are no numbers are taken out of tiles in which rows see different keys.
#include "tree_attention.cuh"

namespace srlm {
namespace tree {

constexpr int S_KEYS = 32, S_WARPS = 4, S_OWN = 8, S_THREADS = 32 * S_WARPS;

__host__ __device__ inline int simt_ld(int hd) { return (hd + 3) / 4 * 4 + 4; }      // rows 16 bytes apart in the banks
template <int KEY_WARPS>
struct SimtForm {
  static constexpr int ROWS = S_OWN * S_WARPS / KEY_WARPS, WK = S_KEYS / KEY_WARPS, PER = S_OWN / KEY_WARPS;      // keys of a warp, rows of a lane
  static size_t smem(int hd) {
    return sizeof(float) * ((size_t)(4 * S_KEYS + ROWS) * simt_ld(hd) + S_WARPS * S_OWN * (WK + 1)) + 3 * S_KEYS * sizeof(long long);
  }
};

// Blocks on an SM: the grid is what runs at once (heads of up to 64, all rows: three, of 168 registers; a fourth wave of blocks that do
// not fit took a quarter longer: 64 rows behind 4,000 keys, 16 entries, 389 | 306 us).
__host__ __device__ constexpr int simt_blocks(int dims, int key_warps) { return dims == 2 ? (key_warps == 1 ? 3 : 4) : dims == 4 ? 2 : 1; }

template <typename T, int DIMS, bool COPY, int KEY_WARPS>
__global__ void __launch_bounds__(S_THREADS, simt_blocks(DIMS, KEY_WARPS)) tree_simt_kernel(const __grid_constant__ Args a) {
  using Form = SimtForm<KEY_WARPS>;
  constexpr int ROWS = Form::ROWS, WK = Form::WK, PER = Form::PER;
  extern __shared__ __align__(16) float tree_sh[];
  const int ld = simt_ld(a.hd), pieces = (a.hd + 3) / 4;
  float* k_sh = tree_sh;                                   // [2][keys][ld]
  float* v_sh = k_sh + 2 * S_KEYS * ld;                    // [2][keys][ld]
  float* q_sh = v_sh + 2 * S_KEYS * ld;                    // [ROWS][ld]
  float* p_sh = q_sh + ROWS * ld;                          // [warps][8][WK] weights
  float* f_sh = p_sh + S_WARPS * S_OWN * WK;               // [warps][8] what the rows' sums so far are multiplied by
  long long* at_sh = reinterpret_cast<long long*>(f_sh + S_WARPS * S_OWN);      // [3][keys]: first element of a key's row; -1: none
  __shared__ int loose_sh;
  const T* q = (const T*)a.q;
  const T* kc = (const T*)a.k_cache;
  const T* vc = (const T*)a.v_cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row_warp = warp / KEY_WARPS, key0 = warp % KEY_WARPS * WK;
  const int key = key0 + lane % WK, rows0 = row_warp * S_OWN + lane / WK * PER;         // the lane's key, and first row, for the scores
  const int g = a.g;
  pdl_wait();
  pdl_trigger();
  Walk<ROWS, S_KEYS> walk;
  walk.init(a, blockIdx.x == 0);
  Piece w;
  if (threadIdx.x == 0) leave_no_unit(a);
  while (walk.next(a, w)) {
    if (threadIdx.x == 0) leave_unit(a, walk, w);
    const Entry& x = w.x;
    const int r0 = w.block * ROWS, rows = min(ROWS, x.q_len * g - r0), tiles = w.tile_hi - w.tile_lo;
    const int* table = a.block_table + (size_t)w.e * a.table_stride;
    const int first_key = a.window > 0 ? max(0, x.start - a.window + 1) : 0;
    auto locate = [&](int t) {
      if (tid < S_KEYS) {
        const int j = (w.tile_lo + t) * S_KEYS + tid;
        at_sh[t % 3 * S_KEYS + tid] = t < tiles && j >= first_key && j < x.kv_len ? row_of_key(a, table, j, w.kvh) * a.hd : -1;
      }
    };
    auto fetch = [&](int t) {
      if (t < tiles) {
        float* kd = k_sh + (t & 1) * S_KEYS * ld;
        float* vd = v_sh + (t & 1) * S_KEYS * ld;
        for (int i = tid; i < S_KEYS * pieces; i += S_THREADS) {
          const int kk = i / pieces, c = (i - kk * pieces) * 4;
          const long long row = at_sh[t % 3 * S_KEYS + kk], at = row < 0 ? 0 : row + c;
          if constexpr (COPY) {
            const unsigned ka = (unsigned)__cvta_generic_to_shared(kd + kk * ld + c);
            const unsigned va = (unsigned)__cvta_generic_to_shared(vd + kk * ld + c);
            const int bytes = row < 0 ? 0 : 16;            // 0: zeros
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ka), "l"(kc + at), "r"(bytes) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(va), "l"(vc + at), "r"(bytes) : "memory");
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool in = row >= 0 && c + e < a.hd;
              kd[kk * ld + c + e] = in ? to_float(kc[at + e]) : 0.f;
              vd[kk * ld + c + e] = in ? to_float(vc[at + e]) : 0.f;
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    locate(0);
    locate(1);
    if (tid == 0) loose_sh = 0;
    if (COPY && ((uintptr_t)a.q & 15) == 0) {              // (in the first tile's group: there before it is read)
      for (int i = tid; i < ROWS * pieces; i += S_THREADS) {
        const int row = i / pieces, c = (i - row * pieces) * 4, r = r0 + row;
        const bool there = row < rows;
        const unsigned at = (unsigned)__cvta_generic_to_shared(q_sh + row * ld + c);
        const T* src = there ? q + ((size_t)(x.q0 + r / g) * a.nq + w.kvh * g + r % g) * a.hd + c : q;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(src), "r"(there ? 16 : 0) : "memory");
      }
    } else {
#pragma unroll 8
      for (int i = tid; i < ROWS * ld; i += S_THREADS) {
        const int row = i / ld, d = i - row * ld, r = r0 + row;
        q_sh[i] = row < rows && d < a.hd ? to_float(q[((size_t)(x.q0 + r / g) * a.nq + w.kvh * g + r % g) * a.hd + d]) : 0.f;
      }
    }
    __syncthreads();
    fetch(0);

    float acc[S_OWN][DIMS], m[PER], l[PER];
#pragma unroll
    for (int o = 0; o < S_OWN; ++o)
#pragma unroll
      for (int i = 0; i < DIMS; ++i) acc[o][i] = 0.f;
#pragma unroll
    for (int o = 0; o < PER; ++o) m[o] = -CUDART_INF_F, l[o] = 0.f;
    const bool live = row_warp * S_OWN < rows;             // (none of the warp's rows is one: it only copies)
    float* p_own = p_sh + warp * S_OWN * WK;
    float* f_own = f_sh + warp * S_OWN;
    for (int t = 0; t < tiles; ++t) {
      const int j0 = (w.tile_lo + t) * S_KEYS;
      fetch(t + 1);
      locate(t + 2);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      // every row sees every key of a tile between the window's last edge and the drafted tokens
      const bool plain = j0 + S_KEYS <= x.start && (a.window <= 0 || j0 >= x.kv_len - a.window);
      if (!plain) {
        bool loose = false;
        for (int i = tid; i < S_KEYS * pieces; i += S_THREADS) {
          float4* p = reinterpret_cast<float4*>(v_sh + ((t & 1) * S_KEYS + i / pieces) * ld + i % pieces * 4);
          float4 v = *p;
          if (take_loose(v)) {
            *p = v;
            loose = true;
          }
        }
        if (loose) loose_sh = 1;
        __syncthreads();
      }
      if (live) {
        const float4* kp = reinterpret_cast<const float4*>(k_sh + ((t & 1) * S_KEYS + key) * ld);
        const float4* qp = reinterpret_cast<const float4*>(q_sh + rows0 * ld);
        float2 s[PER];
#pragma unroll
        for (int o = 0; o < PER; ++o) s[o] = make_float2(0.f, 0.f);
#pragma unroll 2
        for (int c = 0; c < pieces; ++c) {
          const float4 k = kp[c];
#pragma unroll
          for (int o = 0; o < PER; ++o) {
            const float4 v = qp[o * (ld / 4) + c];
            s[o] = fma2(make_float2(v.x, v.y), make_float2(k.x, k.y), s[o]);
            s[o] = fma2(make_float2(v.z, v.w), make_float2(k.z, k.w), s[o]);
          }
        }
        unsigned seen = rows0 < rows ? (1u << min(PER, rows - rows0)) - 1u : 0u;       // a bit a row
        if (!plain) {
          Sight<1> sight[PER];                             // (all words in flight at once)
          int lo[PER];
#pragma unroll
          for (int o = 0; o < PER; ++o) {
            const int token = x.q0 + (r0 + min(rows0 + o, rows - 1)) / g;
            sight[o].words(a, token, j0, x.start);
            lo[o] = first_key_of(a, token, x.start, x.kv_len);
          }
#pragma unroll
          for (int o = 0; o < PER; ++o) {
            uint32_t bits[1];
            sight[o].bits(bits, j0, x.start, x.kv_len, lo[o]);
            if (!((bits[0] >> key) & 1)) seen &= ~(1u << o);
          }
        }
#pragma unroll
        for (int o = 0; o < PER; ++o) {
          const bool sees = (seen >> o) & 1;
          const float v = sees ? (s[o].x + s[o].y) * a.scale_log2 : -CUDART_INF_F;
          float top = v;
#pragma unroll
          for (int b = WK / 2; b > 0; b >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
          top = fmaxf(top, m[o]);
          const float base = top == -CUDART_INF_F ? 0.f : top;
          const float f = exp2f(m[o] - base), p = exp2f(v - base);
          l[o] = l[o] * f + p;                             // (the lane's own keys; the lanes add up at the end)
          m[o] = top;
          p_own[(lane / WK * PER + o) * WK + lane % WK] = p;
          if (lane % WK == 0) f_own[lane / WK * PER + o] = f;
        }
        __syncwarp();
#pragma unroll
        for (int o = 0; o < S_OWN; ++o) {
          const float f = f_own[o];
#pragma unroll
          for (int i = 0; i < DIMS; ++i) acc[o][i] *= f;
        }
        const float* vp = v_sh + ((t & 1) * S_KEYS + key0) * ld + lane;
#pragma unroll 1
        for (int jj = 0; jj < WK; jj += 4) {
          float v[4][DIMS];
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < DIMS; ++i) v[e][i] = lane + 32 * i < ld ? vp[(jj + e) * ld + 32 * i] : 0.f;
#pragma unroll
          for (int o = 0; o < S_OWN; ++o) {
            const float4 p4 = *reinterpret_cast<const float4*>(p_own + o * WK + jj);
            const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < DIMS; ++i) acc[o][i] = fmaf(p[e], v[e][i], acc[o][i]);
          }
        }
      }
      __syncthreads();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int o = 0; o < PER; ++o)
#pragma unroll
      for (int b = WK / 2; b > 0; b >>= 1) l[o] += __shfl_xor_sync(0xffffffffu, l[o], b);
    // the rows' references and sums through shared memory: a lane has dimensions from here on
    float2* ml_sh = reinterpret_cast<float2*>(p_sh);       // [warps][8]
    __syncwarp();
    if (lane % WK == 0)
#pragma unroll
      for (int o = 0; o < PER; ++o) ml_sh[warp * S_OWN + lane / WK * PER + o] = make_float2(m[o], l[o]);
    float* o_sh = k_sh;                                    // [warps][8][ld], of the warps of the later keys
    if (KEY_WARPS > 1 && warp % KEY_WARPS)
#pragma unroll
      for (int o = 0; o < S_OWN; ++o)
#pragma unroll
        for (int i = 0; i < DIMS; ++i)
          if (lane + 32 * i < ld) o_sh[(warp * S_OWN + o) * ld + lane + 32 * i] = acc[o][i];
    __syncthreads();
    if (live && warp % KEY_WARPS == 0) {
      const bool whole = w.begins && w.ends;
      const size_t slab = slab_of(blockIdx.x, w.begins);
#pragma unroll
      for (int o = 0; o < S_OWN; ++o) {
        const int row = row_warp * S_OWN + o, r = r0 + row;
        if (row >= rows) continue;
        float M = -CUDART_INF_F, L = 0.f;
#pragma unroll
        for (int k = 0; k < KEY_WARPS; ++k) M = fmaxf(M, ml_sh[(warp + k) * S_OWN + o].x);
        const float base = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
        for (int k = 0; k < KEY_WARPS; ++k) {
          const float2 ml = ml_sh[(warp + k) * S_OWN + o];
          const float f = exp2f(ml.x - base);
          L += f * ml.y;
#pragma unroll
          for (int i = 0; i < DIMS; ++i) {
            const float v = k == 0 ? acc[o][i] : lane + 32 * i < ld ? o_sh[((warp + k) * S_OWN + o) * ld + lane + 32 * i] : 0.f;
            acc[o][i] = k == 0 ? f * v : acc[o][i] + f * v;
          }
        }
        if (whole) {
          T* dst = (T*)a.out + ((size_t)(x.q0 + r / g) * a.nq + w.kvh * g + r % g) * a.hd;
          const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
          for (int i = 0; i < DIMS; ++i)
            if (lane + 32 * i < a.hd) dst[lane + 32 * i] = from_float<T>(acc[o][i] * inv);
        } else {
          if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + (slab * ROWS + row) * 2) = make_float2(M, L);
#pragma unroll
          for (int i = 0; i < DIMS; ++i)
            if (lane + 32 * i < a.hd) a.part_o[(slab * a.hd + lane + 32 * i) * ROWS + row] = acc[o][i];
        }
      }
    }
    __syncthreads();                                       // before the next piece's places and rows
    if (loose_sh) {                                        // (what a row sees of them, on top of the rest: that may hold some too)
      const bool whole = w.begins && w.ends;
      const size_t slab = slab_of(blockIdx.x, w.begins);
      for (int i = tid; i < rows * a.hd; i += S_THREADS) {
        const int row = i / a.hd, d = i - row * a.hd, r = r0 + row;
        const float v = loose_values<T, S_KEYS>(a, x.start, x.kv_len, table, w.kvh, x.q0 + r / g, d, w.tile_lo, w.tile_hi);
        if (isfinite(v)) continue;
        T* dst = (T*)a.out + ((size_t)(x.q0 + r / g) * a.nq + w.kvh * g + r % g) * a.hd + d;
        if (whole) *dst = from_float<T>(to_float(*dst) + v);
        else a.part_o[(slab * a.hd + d) * ROWS + row] += v;
      }
      __syncthreads();
    }
  }
}

// Warps along the keys: by the rows that an entry has at most (8 KV heads of 64, 8 entries behind 2,000 keys, us, four | two | one:
// 8 rows 26.6 | 27.6 | 33.5, 16 rows 49.4 | 37.0 | 41.7, 24 rows 54.0 | 53.5 | 51.6).
static int key_warps(int max_rows) { return max_rows <= 8 ? 4 : max_rows <= 16 ? 2 : 1; }

Form simt_form(int hd, int max_rows, int sms) {
  return Form{simt_blocks(hd <= 64 ? 2 : hd <= 128 ? 4 : 8, key_warps(max_rows)) * sms, S_OWN * S_WARPS / key_warps(max_rows), S_KEYS};
}

template <typename T, int DIMS, bool COPY, int KEY_WARPS>
static int run_form(const Args& a, int blocks, cudaStream_t stream) {
  const int smem = (int)SimtForm<KEY_WARPS>::smem(a.hd), most = (int)SimtForm<KEY_WARPS>::smem(32 * DIMS);
  static std::atomic<bool> have[64];
  const cudaError_t e = allow_smem((const void*)tree_simt_kernel<T, DIMS, COPY, KEY_WARPS>, most, have);
  if (e != cudaSuccess) return refuse((int)e, "tree_attention: cannot get %d bytes of shared memory", most);
  launch_pdl(tree_simt_kernel<T, DIMS, COPY, KEY_WARPS>, dim3(blocks), dim3(S_THREADS), smem, stream, a);
  launch_merge<T, SimtForm<KEY_WARPS>::ROWS, S_KEYS>(a, blocks, stream);
  return launched();
}
template <typename T, int DIMS, bool COPY>
static int run_rows(const Args& a, int max_rows, int sms, cudaStream_t stream) {
  const int blocks = simt_form(a.hd, max_rows, sms).blocks;
  switch (key_warps(max_rows)) {
    case 4: return run_form<T, DIMS, COPY, 4>(a, blocks, stream);
    case 2: return run_form<T, DIMS, COPY, 2>(a, blocks, stream);
    default: return run_form<T, DIMS, COPY, 1>(a, blocks, stream);
  }
}
template <typename T, bool COPY>
static int run_dims(const Args& a, int max_rows, int sms, cudaStream_t stream) {
  if (a.hd <= 64) return run_rows<T, 2, COPY>(a, max_rows, sms, stream);
  if (a.hd <= 128) return run_rows<T, 4, COPY>(a, max_rows, sms, stream);
  return run_rows<T, 8, COPY>(a, max_rows, sms, stream);
}
int run_simt(const Args& a, int dtype, int max_rows, int sms, cudaStream_t stream) {
  if (dtype == DT_BF16) return run_dims<bf16, false>(a, max_rows, sms, stream);
  if (a.hd % 4 == 0 && ((uintptr_t)a.k_cache | (uintptr_t)a.v_cache) % 16 == 0) return run_dims<float, true>(a, max_rows, sms, stream);
  return run_dims<float, false>(a, max_rows, sms, stream);
}

}  // namespace tree
}  // namespace srlm
