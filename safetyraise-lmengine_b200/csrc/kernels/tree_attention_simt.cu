// Attention for drafted tokens in float32 arithmetic: the float32 path, and bfloat16 heads whose size the tensor-core forms
// do not take.  What a row sees and how the work is divided: tree_attention.cuh.
//
// A block walks its pieces' keys in tiles of 32 for 32 rows.  A tile's keys and values are copied to shared memory once for
// all rows, the next tile in flight under the current one (float32 rows of whole 16-byte pieces; others are read and
// converted).  Each of the four warps owns eight rows: for the scores a lane is a key, so that a row's maximum and sum are
// warp reductions; for the outputs a lane holds the dimensions lane + 32 i, so that nothing but the weights passes through
// shared memory.  Bound by the FMAs' operands from shared memory (a 16-byte read feeds 32 of them at best).
// A masked key's weight is an exact zero and its value is not multiplied: what stands in a place that a row does not see
// never reaches it.
#include <type_traits>

#include "tree_attention.cuh"

namespace srlm {
namespace tree {

constexpr int S_ROWS = 32, S_KEYS = 32, S_WARPS = 4, S_OWN = S_ROWS / S_WARPS, S_THREADS = 32 * S_WARPS;

__host__ __device__ inline int simt_ld(int hd) { return (hd + 3) / 4 * 4 + 4; }      // rows 16 bytes apart in the banks
static size_t simt_smem(int hd) { return sizeof(float) * ((size_t)(4 * S_KEYS + S_ROWS) * simt_ld(hd) + S_ROWS * S_KEYS); }

template <typename T, int DIMS, bool COPY>
__global__ void __launch_bounds__(S_THREADS) tree_simt_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(16) float tree_sh[];
  const int ld = simt_ld(a.hd), pieces = (a.hd + 3) / 4;
  float* k_sh = tree_sh;                           // [2][keys][ld]
  float* v_sh = k_sh + 2 * S_KEYS * ld;            // [2][keys][ld]
  float* q_sh = v_sh + 2 * S_KEYS * ld;            // [rows][ld]
  float* p_sh = q_sh + S_ROWS * ld;                // [rows][keys]
  const T* q = (const T*)a.q;
  const T* kc = (const T*)a.k_cache;
  const T* vc = (const T*)a.v_cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = a.g;
  pdl_wait();
  pdl_trigger();
  Walk<S_ROWS, S_KEYS> walk;
  walk.init(a, blockIdx.x == 0);
  Piece w;
  if (threadIdx.x == 0) leave_no_unit(a);
  while (walk.next(a, w)) {
    if (threadIdx.x == 0) leave_unit(a, walk, w);
    const Entry& x = w.x;
    const int rows = min(S_ROWS, x.q_len * g - w.block * S_ROWS), r0 = w.block * S_ROWS;
    const int* table = a.block_table + (size_t)w.e * a.table_stride;
    const int first_key = a.window > 0 ? max(0, x.start - a.window + 1) : 0;
    auto fetch = [&](int tile, int stage) {
      float* kd = k_sh + stage * S_KEYS * ld;
      float* vd = v_sh + stage * S_KEYS * ld;
      for (int i = tid; i < S_KEYS * pieces; i += S_THREADS) {
        const int key = i / pieces, c = (i - key * pieces) * 4, j = tile * S_KEYS + key;
        const bool there = j >= first_key && j < x.kv_len;
        const long long at = there ? row_of_key(a, table, j, w.kvh) * a.hd + c : 0;
        if constexpr (COPY) {
          const unsigned ka = (unsigned)__cvta_generic_to_shared(kd + key * ld + c);
          const unsigned va = (unsigned)__cvta_generic_to_shared(vd + key * ld + c);
          const int bytes = there ? 16 : 0;        // 0: zeros
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ka), "l"(kc + at), "r"(bytes) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(va), "l"(vc + at), "r"(bytes) : "memory");
        } else {
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            const bool in = there && c + i4 < a.hd;
            kd[key * ld + c + i4] = in ? to_float(kc[at + i4]) : 0.f;
            vd[key * ld + c + i4] = in ? to_float(vc[at + i4]) : 0.f;
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = tid; i < S_ROWS * ld; i += S_THREADS) {
      const int row = i / ld, d = i - row * ld, r = r0 + row;
      q_sh[i] = row < rows && d < a.hd ? to_float(q[((size_t)(x.q0 + r / g) * a.nq + w.kvh * g + r % g) * a.hd + d]) : 0.f;
    }
    fetch(w.tile_lo, 0);

    float acc[S_OWN][DIMS], m[S_OWN], l[S_OWN];
#pragma unroll
    for (int o = 0; o < S_OWN; ++o) {
      m[o] = -CUDART_INF_F;
      l[o] = 0.f;
#pragma unroll
      for (int i = 0; i < DIMS; ++i) acc[o][i] = 0.f;
    }
    const int own = min(S_OWN, rows - warp * S_OWN);           // rows of this warp (none: it only copies)
    for (int tile = w.tile_lo; tile < w.tile_hi; ++tile) {
      const int stage = (tile - w.tile_lo) & 1, j0 = tile * S_KEYS;
      if (tile + 1 < w.tile_hi) fetch(tile + 1, stage ^ 1);
      else asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      if (own > 0) {
        const float* kp = k_sh + (stage * S_KEYS + lane) * ld;
        const float* qp = q_sh + warp * S_OWN * ld;
        float s[S_OWN];
#pragma unroll
        for (int o = 0; o < S_OWN; ++o) s[o] = 0.f;
        for (int c = 0; c < pieces; ++c) {
          const float4 k = *reinterpret_cast<const float4*>(kp + 4 * c);
#pragma unroll
          for (int o = 0; o < S_OWN; ++o) {
            const float4 v = *reinterpret_cast<const float4*>(qp + o * ld + 4 * c);
            s[o] = fmaf(v.x, k.x, s[o]);
            s[o] = fmaf(v.y, k.y, s[o]);
            s[o] = fmaf(v.z, k.z, s[o]);
            s[o] = fmaf(v.w, k.w, s[o]);
          }
        }
        // every row sees every key of a tile between the window's last edge and the drafted tokens
        const bool plain = j0 + S_KEYS <= x.start && (a.window <= 0 || j0 >= x.kv_len - a.window);
        bool all = plain;
#pragma unroll
        for (int o = 0; o < S_OWN; ++o) {
          if (o < own) {
            bool sees = true;
            if (!plain) {
              const int t = x.q0 + (r0 + warp * S_OWN + o) / g;
              Sight<1> sight;
              uint32_t bits[1];
              sight.words(a, t, j0, x.start);
              sight.bits(bits, j0, x.start, x.kv_len, first_key_of(a, t, x.start));
              sees = (bits[0] >> lane) & 1;
            }
            const float v = sees ? s[o] * a.scale_log2 : -CUDART_INF_F;
            const float m_new = fmaxf(m[o], warp_max(v));
            const float base = m_new == -CUDART_INF_F ? 0.f : m_new;
            const float alpha = exp2f(m[o] - base), p = exp2f(v - base);
            l[o] = l[o] * alpha + warp_sum(p);
            m[o] = m_new;
#pragma unroll
            for (int i = 0; i < DIMS; ++i) acc[o][i] *= alpha;
            p_sh[(warp * S_OWN + o) * S_KEYS + lane] = p;
          } else {
            p_sh[(warp * S_OWN + o) * S_KEYS + lane] = 0.f;
          }
        }
        __syncwarp();
        const float* vp = v_sh + stage * S_KEYS * ld + lane;
        auto add = [&](auto tested) {
#pragma unroll 1
          for (int jj = 0; jj < S_KEYS; jj += 4) {
            float v[4][DIMS];
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < DIMS; ++i) v[e][i] = lane + 32 * i < ld ? vp[(jj + e) * ld + 32 * i] : 0.f;
#pragma unroll
            for (int o = 0; o < S_OWN; ++o) {
              const float4 p4 = *reinterpret_cast<const float4*>(p_sh + (warp * S_OWN + o) * S_KEYS + jj);
              const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!decltype(tested)::value || p[e] != 0.f)
#pragma unroll
                  for (int i = 0; i < DIMS; ++i) acc[o][i] = fmaf(p[e], v[e][i], acc[o][i]);
            }
          }
        };
        if (all) add(std::false_type{}); else add(std::true_type{});
      }
      __syncthreads();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    const bool whole = w.begins && w.ends;
    const size_t slab = slab_of(blockIdx.x, w.begins);
#pragma unroll
    for (int o = 0; o < S_OWN; ++o) {
      if (o >= own) continue;
      const int row = warp * S_OWN + o, r = r0 + row;
      if (whole) {
        T* dst = (T*)a.out + ((size_t)(x.q0 + r / g) * a.nq + w.kvh * g + r % g) * a.hd;
        const float inv = l[o] == 0.f ? 0.f : 1.f / l[o];
#pragma unroll
        for (int i = 0; i < DIMS; ++i)
          if (lane + 32 * i < a.hd) dst[lane + 32 * i] = from_float<T>(acc[o][i] * inv);
      } else {
        if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + (slab * S_ROWS + row) * 2) = make_float2(m[o], l[o]);
#pragma unroll
        for (int i = 0; i < DIMS; ++i)
          if (lane + 32 * i < a.hd) a.part_o[(slab * a.hd + lane + 32 * i) * S_ROWS + row] = acc[o][i];
      }
    }
  }
}

Form simt_form(int hd, int sms) { return Form{(hd <= 64 ? 4 : hd <= 128 ? 2 : 1) * sms, S_ROWS, S_KEYS}; }

template <typename T, int DIMS, bool COPY>
static int run_form(const Args& a, int sms, cudaStream_t stream) {
  const int smem = (int)simt_smem(a.hd), blocks = simt_form(a.hd, sms).blocks;
  static std::atomic<int> have[64];
  const cudaError_t e = allow_smem((const void*)tree_simt_kernel<T, DIMS, COPY>, smem, have);
  if (e != cudaSuccess) return refuse((int)e, "tree_attention: cannot get %d bytes of shared memory", smem);
  launch_pdl(tree_simt_kernel<T, DIMS, COPY>, dim3(blocks), dim3(S_THREADS), smem, stream, a);
  launch_merge<T, S_ROWS>(a, blocks, stream);
  return launched();
}
template <typename T, bool COPY>
static int run_dims(const Args& a, int sms, cudaStream_t stream) {
  if (a.hd <= 64) return run_form<T, 2, COPY>(a, sms, stream);
  if (a.hd <= 128) return run_form<T, 4, COPY>(a, sms, stream);
  return run_form<T, 8, COPY>(a, sms, stream);
}
int run_simt(const Args& a, int dtype, int sms, cudaStream_t stream) {
  if (dtype == DT_BF16) return run_dims<bf16, false>(a, sms, stream);
  if (a.hd % 4 == 0 && ((uintptr_t)a.k_cache | (uintptr_t)a.v_cache) % 16 == 0) return run_dims<float, true>(a, sms, stream);
  return run_dims<float, false>(a, sms, stream);
}

}  // namespace tree
}  // namespace srlm
