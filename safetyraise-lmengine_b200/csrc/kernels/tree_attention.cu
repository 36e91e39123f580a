// The entry of attention for drafted tokens: checks, and which form takes a call.
#include <algorithm>

#include "tree_attention.cuh"

using namespace srlm;

// tcgen05 wherever it takes the sizes, at any number of rows (8 KV heads of 128, pages of 16, us, tcgen05 | warp level: 8 rows behind
// 200 keys 12.0 | 13.0, 8 entries of 16 rows behind 16,000 76 | 105, of 96 rows 84 | 269).
enum Kind { SIMT, MMA, TCGEN05 };
static Kind kind_of(int dtype, int hd, int page_size) {
  if (dtype != DT_BF16 || !tree::mma_takes(hd)) return SIMT;
  return tree::tcgen05_takes(hd, page_size) ? TCGEN05 : MMA;
}
static tree::Form form_of(Kind kind, int hd, int max_rows, int sms) {
  return kind == TCGEN05 ? tree::tcgen05_form(sms) : kind == MMA ? tree::mma_form(hd, max_rows, sms) : tree::simt_form(hd, max_rows, sms);
}

// float32 words of workspace that srlm_tree_attention wants for these sizes, or -1 where it refuses them.
extern "C" long long srlm_tree_attention_workspace(int dtype, int nq, int nkv, int hd, int page_size, int max_q_len, int sms) {
  if ((dtype != DT_F32 && dtype != DT_BF16) || nq <= 0 || nkv <= 0 || nkv > 65535 || nq % nkv || hd <= 0 || hd > 256 || page_size <= 0 ||
      max_q_len <= 0 || sms <= 0 || (long long)max_q_len * (nq / nkv) > (1 << 24)) {
    refuse(ST_BAD_SIZE, "tree_attention: dtype=%d nq=%d nkv=%d hd=%d page_size=%d max_q_len=%d (needs nq %% nkv == 0, hd <= 256)",
           dtype, nq, nkv, hd, page_size, max_q_len);
    return -1;
  }
  const int max_rows = max_q_len * (nq / nkv);
  const tree::Form f = form_of(kind_of(dtype, hd, page_size), hd, max_rows, sms);
  return 2ll * f.blocks * f.rows * (hd + 2) + 4ll * f.blocks;
}

// q, out [T, nq, hd]; caches [num_pages, nkv, page_size, hd]; block_table [n, table_stride]; cu_q [n + 1]; kv_lens [n]; mask
// [T, words]; positions [T], or null without a window.  max_q_len: no entry has more tokens.  work: as above says.
// launches (a host address, or null): how many kernels the call launched.
extern "C" int srlm_tree_attention(const void* q, const void* k_cache, const void* v_cache, void* out, int dtype, long long num_pages,
                                   const int* block_table, int table_stride, const int* cu_q, const int* kv_lens, const int* mask,
                                   int words, const int* positions, int n, int T, int nq, int nkv, int hd, int page_size, float scale,
                                   int window, int max_q_len, float* work, int sms, int* err_flag, int* launches, cudaStream_t stream) {
  if (launches) *launches = 0;
  if (n <= 0 || T <= 0) return ST_OK;
  if (srlm_tree_attention_workspace(dtype, nq, nkv, hd, page_size, max_q_len, sms) < 0) return ST_BAD_SIZE;
  if (words <= 0 || table_stride <= 0 || num_pages <= 0 || num_pages > 0x7fffffff || window < 0 || (window > 0 && !positions) || !(scale > 0.f) || !work ||
      !err_flag)
    return refuse(ST_BAD_SIZE, "tree_attention: words=%d table_stride=%d num_pages=%lld window=%d scale=%g (a window needs the positions, a "
                  "scale is positive)", words, table_stride, num_pages, window, (double)scale);
  const int max_rows = max_q_len * (nq / nkv);
  const Kind kind = kind_of(dtype, hd, page_size);
  const tree::Form f = form_of(kind, hd, max_rows, sms);
  // the list of all units' tiles is counted in 31 bits, and so are an entry's keys with a tile to spare
  const double units = (double)n * nkv * ((double)max_q_len * (nq / nkv) / f.rows + 1), tiles = (double)table_stride * page_size / f.keys + 1;
  if (units * tiles > 2147483647.0 || (long long)table_stride * page_size > (1 << 30))
    return refuse(ST_BAD_SIZE, "tree_attention: %d entries of up to %d tokens and %d pages are more work than a call takes", n, max_q_len,
                  table_stride);
  float* ml = work + 2ll * f.blocks * f.rows * hd;      // (sizes are multiples of 16 bytes)
  tree::Args a{q, k_cache, v_cache, out, block_table, table_stride, cu_q, kv_lens, mask, words, std::min(max_q_len, 32 * words), positions, n, T,
               nq, nkv, nq / nkv, hd, page_size, (int)num_pages, scale * 1.4426950408889634f,
               2.f * hd * (dtype == DT_F32 ? 4 : 2), window, 1, err_flag, work,
               ml, reinterpret_cast<int4*>(ml + 4ll * f.blocks * f.rows)};
  // A unit of few tiles by the block table's width is not divided: its last tiles take less than the merge and its launch (3.5 us of the
  // host's time besides; us, divided | not: tcgen05 behind 300 keys 12.6 | 10.6, 500 12.0 | 11.0, 800 13.1 | 14.4; warp level behind 120
  // 9.4 | 8.1, 200 9.8 | 10.0, 300 10.0 | 11.3; float32 behind 120 11.8 | 13.5).  Else parts and
  // shares have two tiles at least (8 KV heads, 16 or 32 rows, us, 1 | 2 | 4: tcgen05 behind 200 keys 12.3 | 10.6 | 10.5, behind 2,000
  // 16.6 | 14.7 | 15.8; warp level 11.1 | 12.3 | 15.4 and 18.0 | 15.0 | 15.1; float32 13.3 | 15.0 | 18.7 and 22.5 | 20.4 | 22.0).
  const long long keys = (long long)table_stride * page_size, most = (keys + f.keys - 1) / f.keys;
  a.least_tiles = most <= (kind == TCGEN05 ? 6 : kind == MMA ? 4 : 2) ? (int)most : 2;
  if (launches) *launches = tree::merges(a, f.blocks, f.rows, f.keys) ? 2 : 1;
  if (kind == SIMT) return tree::run_simt(a, dtype, max_rows, sms, stream);
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) % 16)
    return refuse(ST_BAD_ALIGN, "tree_attention: bfloat16 tensors start on 16-byte boundaries");
  return kind == TCGEN05 ? tree::run_tcgen05(a, sms, stream) : tree::run_mma(a, max_rows, sms, stream);
}
