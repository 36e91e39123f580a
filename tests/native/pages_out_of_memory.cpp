// Forks and compactions whose allocations fail, one after another: what the C API calls "nothing changed" has to be so.
#include <cstdio>
#include <cstdlib>
#include <new>
#include <vector>

#include "runtime_c_api.h"

static long left = -1;      // allocations until one fails; -1: none does

void* operator new(size_t n) {
  if (left == 0) throw std::bad_alloc();
  if (left > 0) --left;
  if (void* p = std::malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, size_t) noexcept { std::free(p); }

static std::vector<int> tables(void* c) {
  std::vector<int> all;
  int32_t pages[64];
  for (int g = 0; g < 3; ++g)
    for (int s = 0; s < 4; ++s) {
      const int n = srlm_cache_table(c, g, s, pages, 64);
      all.push_back(n);
      for (int i = 0; i < n; ++i) all.push_back(pages[i]);
    }
  for (int g = 0; g < 3; ++g) all.push_back(srlm_cache_free_pages(c, g));
  return all;
}

#define CHECK(x)                                            \
  do {                                                      \
    if (!(x)) {                                             \
      std::printf("line %d, allocation %ld: %s\n", __LINE__, k, #x); \
      return 1;                                             \
    }                                                       \
  } while (0)

int main() {
  const int kinds[3] = {0, 0, 0}, sizes[3] = {4, 4, 4}, pages[3] = {20, 20, 20}, none[3] = {0, 0, 0};
  int32_t copies[3 * 60];
  for (int what = 0; what < 3; ++what) {
    bool done = false;
    for (long k = 0; !done; ++k) {
      void* c = srlm_cache_create(4, 3, kinds, sizes, pages, none, none);
      const int a = srlm_cache_open(c), b = srlm_cache_open(c);
      CHECK(srlm_cache_reserve(c, a, 16) == 1 && srlm_cache_commit(c, a, 16) == 0);
      CHECK(srlm_cache_reserve(c, b, 16) == 1 && srlm_cache_commit(c, b, 16) == 0);
      int n = 0;
      const int f = srlm_cache_fork(c, b, 16, copies, 60, &n);      // shares b's four pages
      CHECK(f >= 0);
      CHECK(srlm_cache_close(c, a) == 0);
      if (what == 1) CHECK(srlm_cache_open(c) == a);                // the fork's slot has held no table before
      const std::vector<int> was = tables(c);
      left = k;
      const int r = what == 0 ? srlm_cache_compact(c, copies, 60, &n) : what == 1 ? srlm_cache_fork(c, b, 14, copies, 60, &n)
                                                                                  : srlm_cache_unshare(c, b, 14, copies, 60, &n);
      left = -1;
      if (r == -9) {
        CHECK(n == 0);
        CHECK(srlm_cache_audit(c) == 0);
        CHECK(tables(c) == was);
        int slots = 0;
        while (srlm_cache_open(c) >= 0) ++slots;
        CHECK(slots == (what == 1 ? 1 : 2));                        // none was lost
      } else {
        CHECK(k > 0);
        CHECK(r >= 0 && n > 0);
        CHECK(srlm_cache_audit(c) == 0);
        done = true;
      }
      srlm_cache_destroy(c);
    }
  }
  std::printf("ok\n");
  return 0;
}
