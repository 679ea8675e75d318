// Host-side bookkeeping of a paged K/V cache: page tables, lengths and how
// many sequences hold each page (b2_page_pool_*).  No device calls; the
// lowest free page is taken first, so a pool in light use stays compact.
#include <algorithm>
#include <functional>
#include <new>
#include <vector>

#include "b2_internal.hpp"

struct b2_page_pool {
  int32_t page_size = 0, max_pages = 0;
  std::vector<int32_t> ref;                  // holders of each page
  std::vector<int32_t> free_heap;            // min-heap of free pages
  std::vector<std::vector<int32_t>> pages;   // per sequence, in order
  std::vector<int32_t> len;                  // positions per sequence
  std::vector<int32_t> held;                 // released by keep, until settle
};

namespace {

int32_t pages_for(const b2_page_pool* p, int64_t n) { return (int32_t)((n + p->page_size - 1) / p->page_size); }
bool seq_ok(const b2_page_pool* p, int32_t s) { return p && s >= 0 && s < (int32_t)p->pages.size(); }

int32_t take(b2_page_pool* p) {
  std::pop_heap(p->free_heap.begin(), p->free_heap.end(), std::greater<int32_t>());
  const int32_t page = p->free_heap.back();
  p->free_heap.pop_back();
  p->ref[page] = 1;
  return page;
}
void drop(b2_page_pool* p, int32_t page) {
  if (--p->ref[page] == 0) {
    p->free_heap.push_back(page);   // capacity reserved for every page
    std::push_heap(p->free_heap.begin(), p->free_heap.end(), std::greater<int32_t>());
  }
}
int out_of_memory() {
  b2::set_error("page pool: out of host memory");
  return B2_ERR_OOM;
}

}  // namespace

extern "C" {

int b2_page_pool_create(int32_t n_pages, int32_t page_size, int32_t n_seq, int32_t max_pages, b2_page_pool** out) {
  B2_CHECK_ARG(out && n_pages > 0 && n_seq > 0 && max_pages > 0, "page_pool_create arguments");
  B2_CHECK_ARG(page_size >= 1 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
               "page_size must be a power of two up to 256");
  B2_CHECK_ARG((int64_t)max_pages * page_size <= (1 << 30), "page_pool_create: max_pages");
  *out = nullptr;
  try {
    b2_page_pool* p = new b2_page_pool;
    try {
      p->page_size = page_size;
      p->max_pages = max_pages;
      p->ref.assign(n_pages, 0);
      p->free_heap.resize(n_pages);
      for (int32_t i = 0; i < n_pages; ++i) p->free_heap[i] = i;   // ascending: a heap
      p->pages.resize(n_seq);
      p->len.assign(n_seq, 0);
    } catch (...) {
      delete p;
      throw;
    }
    *out = p;
  } catch (const std::bad_alloc&) {
    return out_of_memory();
  }
  return B2_OK;
}

int b2_page_pool_destroy(b2_page_pool* p) {
  delete p;
  return B2_OK;
}

int b2_page_pool_extend(b2_page_pool* p, int32_t seq, int32_t n, int32_t* copy_src, int32_t* copy_dst) {
  B2_CHECK_ARG(seq_ok(p, seq) && n >= 0 && copy_src && copy_dst, "page_pool_extend arguments");
  *copy_src = *copy_dst = -1;
  if (n == 0) return B2_OK;
  std::vector<int32_t>& v = p->pages[seq];
  const int64_t len = (int64_t)p->len[seq] + n;
  if (len > (int64_t)p->max_pages * p->page_size) return B2_NO_KV_SLOT;
  const int32_t want = pages_for(p, len), more = want - (int32_t)v.size();
  const bool copy = p->len[seq] % p->page_size != 0 && p->ref[v.back()] > 1;
  if (more + (copy ? 1 : 0) > (int32_t)p->free_heap.size()) return B2_NO_KV_SLOT;
  try {
    v.reserve(want);
  } catch (const std::bad_alloc&) {
    return out_of_memory();
  }
  if (copy) {
    *copy_src = v.back();
    *copy_dst = take(p);
    drop(p, v.back());
    v.back() = *copy_dst;
  }
  for (int32_t i = 0; i < more; ++i) v.push_back(take(p));
  p->len[seq] = (int32_t)len;
  return B2_OK;
}

int b2_page_pool_fork(b2_page_pool* p, int32_t src, int32_t dst, int32_t n) {
  B2_CHECK_ARG(seq_ok(p, src) && seq_ok(p, dst) && src != dst, "page_pool_fork sequences");
  B2_CHECK_ARG(n >= 0 && n <= p->len[src], "page_pool_fork: n beyond the source");
  B2_CHECK_ARG(p->len[dst] == 0, "page_pool_fork: the destination holds positions");
  const int32_t k = pages_for(p, n);
  try {
    p->pages[dst].assign(p->pages[src].begin(), p->pages[src].begin() + k);
  } catch (const std::bad_alloc&) {
    return out_of_memory();
  }
  for (int32_t page : p->pages[dst]) ++p->ref[page];
  p->len[dst] = n;
  return B2_OK;
}

int b2_page_pool_truncate(b2_page_pool* p, int32_t seq, int32_t n) {
  B2_CHECK_ARG(seq_ok(p, seq) && n >= 0 && n <= p->len[seq], "page_pool_truncate arguments");
  std::vector<int32_t>& v = p->pages[seq];
  const size_t k = (size_t)pages_for(p, n);
  while (v.size() > k) {
    drop(p, v.back());
    v.pop_back();
  }
  p->len[seq] = n;
  return B2_OK;
}

int b2_page_pool_keep(b2_page_pool* p, int32_t seq, const int32_t* keep, int32_t n, int32_t* old_table) {
  B2_CHECK_ARG(seq_ok(p, seq) && n >= 0 && (n == 0 || keep) && old_table, "page_pool_keep arguments");
  for (int32_t i = 0; i < n; ++i)
    B2_CHECK_ARG(keep[i] < p->len[seq] && keep[i] >= (i ? keep[i - 1] + 1 : 0),
                 "page_pool_keep: positions must ascend and lie in the sequence");
  std::vector<int32_t>& v = p->pages[seq];
  int32_t same = 0;   // leading positions that stay where they are
  while (same < n && keep[same] == same) ++same;
  // whole pages of them, and all of the last page when nothing follows it
  const int32_t stay = same == n ? pages_for(p, n) : same / p->page_size;
  const int32_t fresh = pages_for(p, n) - stay;
  if (fresh > (int32_t)p->free_heap.size()) return B2_NO_KV_SLOT;
  try {
    p->held.reserve(p->held.size() + v.size());
  } catch (const std::bad_alloc&) {
    return out_of_memory();
  }
  for (int32_t i = 0; i < p->max_pages; ++i) old_table[i] = i < (int32_t)v.size() ? v[i] : -1;
  for (size_t i = stay; i < v.size(); ++i) p->held.push_back(v[i]);
  v.resize(stay);   // fresh <= pages given up, so the capacity suffices
  for (int32_t i = 0; i < fresh; ++i) v.push_back(take(p));
  p->len[seq] = n;
  return B2_OK;
}

int b2_page_pool_settle(b2_page_pool* p) {
  B2_CHECK_ARG(p, "page_pool_settle");
  for (int32_t page : p->held) drop(p, page);
  p->held.clear();
  return B2_OK;
}

int b2_page_pool_defrag(b2_page_pool* p, int32_t* src, int32_t* dst, int32_t room, int32_t* n) {
  B2_CHECK_ARG(p && n && room >= 0 && (room == 0 || (src && dst)), "page_pool_defrag arguments");
  B2_CHECK_ARG(p->held.empty(), "page_pool_defrag: settle held pages first");
  *n = 0;
  const int32_t total = (int32_t)p->ref.size(), used = total - (int32_t)p->free_heap.size();
  int32_t moves = 0;
  for (int32_t i = used; i < total; ++i) moves += p->ref[i] > 0;
  B2_CHECK_ARG(moves <= room, "page_pool_defrag: more moves than room");
  try {
    std::vector<int32_t> to(total, -1);
    int32_t lo = 0;
    for (int32_t i = used; i < total; ++i) {
      if (p->ref[i] == 0) continue;
      while (p->ref[lo] > 0) ++lo;   // a free page below `used` exists for every used page above it
      to[i] = lo;
      src[*n] = i;
      dst[(*n)++] = lo;
      p->ref[lo] = p->ref[i];
      p->ref[i] = 0;
    }
    for (std::vector<int32_t>& v : p->pages)
      for (int32_t& page : v)
        if (to[page] >= 0) page = to[page];
  } catch (const std::bad_alloc&) {
    return out_of_memory();   // thrown by `to`, before any change
  }
  for (int32_t i = used; i < total; ++i) p->free_heap[i - used] = i;
  return B2_OK;
}

int b2_page_pool_table(const b2_page_pool* p, int32_t seq, int32_t* out, int32_t* length) {
  B2_CHECK_ARG(seq_ok(p, seq), "page_pool_table sequence");
  const std::vector<int32_t>& v = p->pages[seq];
  if (out)
    for (int32_t i = 0; i < p->max_pages; ++i) out[i] = i < (int32_t)v.size() ? v[i] : -1;
  if (length) *length = p->len[seq];
  return B2_OK;
}

int b2_page_pool_free_pages(const b2_page_pool* p, int32_t* n) {
  B2_CHECK_ARG(p && n, "page_pool_free_pages arguments");
  *n = (int32_t)p->free_heap.size();
  return B2_OK;
}

}  // extern "C"
