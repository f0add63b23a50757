// kv_pool.cpp -- host-side page allocator for the paged KV cache.
//
// The reference binds one page_table per dispatch
// (runtime/zig/tests/tsir/real/attention_head256_f16kv/attention_head256_f16kv.wgsl:38,
// consumed by get_kv_pos, :51-63) and leaves its contents to the caller.  This
// pool is that caller for the batched kernels: it owns the free list of
// physical pages and the per-sequence rows of the block table
// ([max_seqs, max_pages_per_seq] int32, -1 = unmapped).  Sequences may share
// pages (fork): a page goes back to the free list with its last reference, and
// make_writable gives a sequence pages of its own before it writes shared ones.
// Pure host code; no C++ exception leaves an entry point.
#include <cstring>
#include <mutex>
#include <new>
#include <vector>

#include "../../include/doe_cuda.h"

struct doe_kv_pool {
  uint32_t num_pages = 0;
  uint32_t page_size = 0;
  uint32_t max_seqs = 0;
  uint32_t max_pages = 0;
  std::vector<int32_t> free_list;           // LIFO stack of free pages
  std::vector<std::vector<int32_t>> pages;  // per sequence, logical order
  std::vector<uint32_t> refs;               // per page, sequences that hold it
  std::mutex mu;
};

namespace {

// An entry point's body: allocation failures become a status.
template <typename F>
int guarded(F&& body) {
  try {
    return body();
  } catch (...) {
    return DOE_ERROR;
  }
}

// Gives back a sequence's pages from logical page `keep` on, last page first.
// free_list has room for every page, so nothing here allocates.
void drop_pages(doe_kv_pool* p, std::vector<int32_t>& row, uint64_t keep) {
  while (row.size() > keep) {
    const int32_t page = row.back();
    row.pop_back();
    if (--p->refs[page] == 0) p->free_list.push_back(page);
  }
}

uint64_t pages_of(const doe_kv_pool* p, uint32_t tokens) {
  return ((uint64_t)tokens + p->page_size - 1) / p->page_size;
}

}  // namespace

extern "C" {

int doe_kv_pool_create(uint32_t num_pages, uint32_t page_size, uint32_t max_seqs,
                       uint32_t max_pages_per_seq, doe_kv_pool** out) {
  if (!out) return DOE_INVALID_ARGUMENT;
  *out = nullptr;
  if (num_pages == 0 || page_size == 0 || max_seqs == 0 || max_pages_per_seq == 0)
    return DOE_INVALID_ARGUMENT;
  if (num_pages > 0x7fffffffu) return DOE_INVALID_ARGUMENT;
  doe_kv_pool* p = nullptr;
  const int rc = guarded([&] {
    p = new doe_kv_pool();
    p->num_pages = num_pages;
    p->page_size = page_size;
    p->max_seqs = max_seqs;
    p->max_pages = max_pages_per_seq;
    p->free_list.reserve(num_pages);
    for (uint32_t i = num_pages; i > 0; --i) p->free_list.push_back((int32_t)(i - 1));
    p->pages.resize(max_seqs);
    p->refs.resize(num_pages, 0);
    return (int)DOE_OK;
  });
  if (rc != DOE_OK) {
    delete p;
    return rc;
  }
  *out = p;
  return DOE_OK;
}

int doe_kv_pool_destroy(doe_kv_pool* pool) {
  if (!pool) return DOE_INVALID_ARGUMENT;
  delete pool;
  return DOE_OK;
}

int doe_kv_pool_reserve(doe_kv_pool* pool, uint32_t seq, uint32_t tokens) {
  if (!pool) return DOE_INVALID_ARGUMENT;
  return guarded([&]() -> int {
    std::lock_guard<std::mutex> lock(pool->mu);
    if (seq >= pool->max_seqs) return DOE_OUT_OF_RANGE;
    const uint64_t need = pages_of(pool, tokens);
    if (need > pool->max_pages) return DOE_OUT_OF_RANGE;
    std::vector<int32_t>& row = pool->pages[seq];
    if (need <= row.size()) return DOE_OK;
    const uint64_t extra = need - row.size();
    if (extra > pool->free_list.size()) return DOE_OUT_OF_RANGE;  // pool exhausted
    row.reserve(need);  // nothing below allocates
    for (uint64_t i = 0; i < extra; ++i) {
      row.push_back(pool->free_list.back());
      pool->free_list.pop_back();
      pool->refs[row.back()] = 1;
    }
    return DOE_OK;
  });
}

int doe_kv_pool_release(doe_kv_pool* pool, uint32_t seq) {
  if (!pool) return DOE_INVALID_ARGUMENT;
  return guarded([&]() -> int {
    std::lock_guard<std::mutex> lock(pool->mu);
    if (seq >= pool->max_seqs) return DOE_OUT_OF_RANGE;
    drop_pages(pool, pool->pages[seq], 0);
    return DOE_OK;
  });
}

int doe_kv_pool_truncate(doe_kv_pool* pool, uint32_t seq, uint32_t tokens) {
  if (!pool) return DOE_INVALID_ARGUMENT;
  return guarded([&]() -> int {
    std::lock_guard<std::mutex> lock(pool->mu);
    if (seq >= pool->max_seqs) return DOE_OUT_OF_RANGE;
    drop_pages(pool, pool->pages[seq], pages_of(pool, tokens));
    return DOE_OK;
  });
}

int doe_kv_pool_fork(doe_kv_pool* pool, uint32_t from, uint32_t to, uint32_t tokens) {
  if (!pool || from == to) return DOE_INVALID_ARGUMENT;
  return guarded([&]() -> int {
    std::lock_guard<std::mutex> lock(pool->mu);
    if (from >= pool->max_seqs || to >= pool->max_seqs) return DOE_OUT_OF_RANGE;
    const std::vector<int32_t>& src = pool->pages[from];
    std::vector<int32_t>& dst = pool->pages[to];
    if (!dst.empty()) return DOE_INVALID_ARGUMENT;
    const uint64_t n = pages_of(pool, tokens);
    if (n > src.size()) return DOE_OUT_OF_RANGE;
    dst.assign(src.begin(), src.begin() + (ptrdiff_t)n);
    for (int32_t page : dst) ++pool->refs[page];
    return DOE_OK;
  });
}

int doe_kv_pool_make_writable(doe_kv_pool* pool, uint32_t seq, uint32_t first_token, uint32_t tokens,
                              int32_t* pairs, uint32_t max_pairs, uint32_t* num_pairs) {
  if (!pool || !num_pairs || (!pairs && max_pairs != 0)) return DOE_INVALID_ARGUMENT;
  *num_pairs = 0;
  return guarded([&]() -> int {
    std::lock_guard<std::mutex> lock(pool->mu);
    if (seq >= pool->max_seqs) return DOE_OUT_OF_RANGE;
    if (tokens == 0) return DOE_OK;
    std::vector<int32_t>& row = pool->pages[seq];
    const uint64_t p0 = first_token / pool->page_size;
    const uint64_t p1 = ((uint64_t)first_token + tokens + pool->page_size - 1) / pool->page_size;
    if (p1 > row.size()) return DOE_OUT_OF_RANGE;
    uint64_t shared = 0;
    for (uint64_t i = p0; i < p1; ++i) shared += pool->refs[row[i]] > 1;
    if (shared > pool->free_list.size()) return DOE_OUT_OF_RANGE;  // pool exhausted
    if (shared > max_pairs) return DOE_INVALID_ARGUMENT;
    uint32_t n = 0;
    for (uint64_t i = p0; i < p1; ++i) {
      const int32_t page = row[i];
      if (pool->refs[page] <= 1) continue;
      const int32_t own = pool->free_list.back();
      pool->free_list.pop_back();
      --pool->refs[page];
      pool->refs[own] = 1;
      row[i] = own;
      pairs[2 * n] = page;
      pairs[2 * n + 1] = own;
      ++n;
    }
    *num_pairs = n;
    return DOE_OK;
  });
}

int doe_kv_pool_compact(doe_kv_pool* pool, int32_t* pairs, uint32_t max_pairs, uint32_t* num_pairs) {
  if (!pool || !num_pairs || (!pairs && max_pairs != 0)) return DOE_INVALID_ARGUMENT;
  *num_pairs = 0;
  return guarded([&]() -> int {
    std::lock_guard<std::mutex> lock(pool->mu);
    const uint32_t live = pool->num_pages - (uint32_t)pool->free_list.size();
    // every live page at or above `live` goes to a free one below it
    std::vector<int32_t> moved(pool->num_pages, -1);
    std::vector<uint32_t> refs(pool->num_pages, 0);
    uint32_t n = 0, hole = 0;
    for (uint32_t page = 0; page < pool->num_pages; ++page) {
      if (pool->refs[page] == 0) continue;
      uint32_t at = page;
      if (page >= live) {
        while (pool->refs[hole] != 0) ++hole;
        at = hole++;
        ++n;
      }
      moved[page] = (int32_t)at;
      refs[at] = pool->refs[page];
    }
    if (n > max_pairs) return DOE_INVALID_ARGUMENT;
    uint32_t k = 0;
    for (uint32_t page = live; page < pool->num_pages; ++page) {
      if (moved[page] < 0) continue;
      pairs[2 * k] = (int32_t)page;
      pairs[2 * k + 1] = moved[page];
      ++k;
    }
    for (std::vector<int32_t>& row : pool->pages)
      for (int32_t& page : row) page = moved[page];
    pool->refs.swap(refs);
    pool->free_list.clear();
    for (uint32_t page = pool->num_pages; page > live; --page) pool->free_list.push_back((int32_t)(page - 1));
    *num_pairs = n;
    return DOE_OK;
  });
}

int doe_kv_pool_page_refs(const doe_kv_pool* pool, uint32_t page, uint32_t* out) {
  if (!pool || !out) return DOE_INVALID_ARGUMENT;
  return guarded([&]() -> int {
    std::lock_guard<std::mutex> lock(const_cast<doe_kv_pool*>(pool)->mu);
    if (page >= pool->num_pages) return DOE_OUT_OF_RANGE;
    *out = pool->refs[page];
    return DOE_OK;
  });
}

int doe_kv_pool_free_pages(const doe_kv_pool* pool, uint32_t* out) {
  if (!pool || !out) return DOE_INVALID_ARGUMENT;
  std::lock_guard<std::mutex> lock(const_cast<doe_kv_pool*>(pool)->mu);
  *out = (uint32_t)pool->free_list.size();
  return DOE_OK;
}

int doe_kv_pool_seq_pages(const doe_kv_pool* pool, uint32_t seq, uint32_t* out) {
  if (!pool || !out) return DOE_INVALID_ARGUMENT;
  std::lock_guard<std::mutex> lock(const_cast<doe_kv_pool*>(pool)->mu);
  if (seq >= pool->max_seqs) return DOE_OUT_OF_RANGE;
  *out = (uint32_t)pool->pages[seq].size();
  return DOE_OK;
}

int doe_kv_pool_block_table(const doe_kv_pool* pool, int32_t* out, uint64_t out_entries) {
  if (!pool || !out) return DOE_INVALID_ARGUMENT;
  std::lock_guard<std::mutex> lock(const_cast<doe_kv_pool*>(pool)->mu);
  const uint64_t total = (uint64_t)pool->max_seqs * pool->max_pages;
  if (out_entries < total) return DOE_INVALID_ARGUMENT;
  for (uint32_t s = 0; s < pool->max_seqs; ++s) {
    int32_t* row = out + (uint64_t)s * pool->max_pages;
    const std::vector<int32_t>& pg = pool->pages[s];
    for (uint32_t i = 0; i < pool->max_pages; ++i) row[i] = i < pg.size() ? pg[i] : -1;
  }
  return DOE_OK;
}

}  // extern "C"
