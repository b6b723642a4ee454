// paged_book.cpp -- which pages of a paged KV cache belong to which sequence:
// reference counts, free pages lowest first, and the lists of page copies that
// forks (copy on write) and compaction ask of exl3p_copy_pages.  Host only.
#include <algorithm>
#include <new>
#include <queue>
#include <vector>

#include "../../include/exl3_paged.h"

namespace {

constexpr exl3_verdict OK{EXL3_OK, ""};
exl3_verdict refuse(int32_t code, const char *why) { return exl3_verdict{code, why}; }

}  // namespace

struct exl3p_book {
  int32_t page, seqs, max_pages;
  std::vector<int32_t> refs;                 // holders of each page
  std::vector<int32_t> table;                // [seqs][max_pages], -1 behind the held ones
  std::vector<int32_t> held;                 // pages of each sequence
  std::priority_queue<int32_t, std::vector<int32_t>, std::greater<int32_t>> free;

  int32_t *row(int32_t seq) { return table.data() + (size_t)seq * max_pages; }
  // free.pop() never allocates; put() may, so the container keeps its capacity
  // for every page from the start
  int32_t take() {
    const int32_t p = free.top();
    free.pop();
    refs[p] = 1;
    return p;
  }
  void put(int32_t p) {
    if (--refs[p] == 0) free.push(p);
  }
  int64_t pages_of(int64_t keys) const { return (keys + page - 1) / page; }
};

extern "C" {

exl3p_book *exl3p_book_open(int32_t pages, int32_t page, int32_t seqs, int32_t max_pages,
                            exl3_verdict *why) {
  exl3_verdict none;
  if (why == nullptr) why = &none;
  *why = OK;
  if (pages <= 0 || seqs <= 0 || max_pages <= 0 || page < 16 || page > 256 ||
      (page & (page - 1)) != 0) {
    *why = refuse(EXL3_UNSUPPORTED, "PagedBookShape: pages, seqs and max_pages above 0, page a "
                                    "power of two from 16 to 256");
    return nullptr;
  }
  if ((int64_t)pages * page > INT32_MAX || (int64_t)max_pages * page > 1 << 30) {
    *why = refuse(EXL3_TOO_LARGE, "PagedBookShape: 2^31 keys or more, or over 2^30 of a sequence");
    return nullptr;
  }
  try {
    auto *b = new exl3p_book;
    try {
      b->page = page, b->seqs = seqs, b->max_pages = max_pages;
      b->refs.assign(pages, 0);
      b->table.assign((size_t)seqs * max_pages, -1);
      b->held.assign(seqs, 0);
      std::vector<int32_t> all(pages);  // ascending: a heap already
      for (int32_t i = 0; i < pages; ++i) all[i] = i;
      b->free = decltype(b->free)(std::greater<int32_t>(), std::move(all));
    } catch (...) {
      delete b;
      throw;
    }
    return b;
  } catch (...) {
    *why = refuse(EXL3_FAILED, "PagedBook: out of host memory");
    return nullptr;
  }
}

void exl3p_book_close(exl3p_book *b) { delete b; }

exl3_verdict exl3p_book_reserve(exl3p_book *b, int32_t seq, int32_t from, int32_t to, int32_t *src,
                                int32_t *dst, int32_t room, int32_t *pairs) {
  if (b == nullptr || pairs == nullptr || room < 0 ||
      (room > 0 && (src == nullptr || dst == nullptr)))
    return refuse(EXL3_FAILED, "PagedBook: a missing argument");
  *pairs = 0;
  if (seq < 0 || seq >= b->seqs) return refuse(EXL3_UNSUPPORTED, "PagedBook: no such sequence");
  if (from < 0 || to < from) return refuse(EXL3_UNSUPPORTED, "PagedBook: keys out of order");
  const int64_t need = b->pages_of(to);
  if (need > b->max_pages)
    return refuse(EXL3_TOO_LARGE, "PagedBook: the sequence's table is full");
  int32_t *t = b->row(seq);
  const int32_t held = b->held[seq];
  const int32_t first = to > from ? from / b->page : (int32_t)need;
  int64_t fresh = std::max<int64_t>(0, need - held), copies = 0;
  for (int64_t i = first; i < std::min<int64_t>(need, held); ++i)
    if (b->refs[t[i]] > 1) {
      ++fresh;
      copies += i * b->page < from;  // keys below `from` live on in the copy
    }
  if (fresh > (int64_t)b->free.size())
    return refuse(EXL3_TOO_LARGE, "PagedBook: no free page is left");
  if (copies > room) return refuse(EXL3_TOO_LARGE, "PagedBook: no room for the pairs to copy");
  for (int64_t i = first; i < std::min<int64_t>(need, held); ++i)
    if (b->refs[t[i]] > 1) {
      const int32_t old = t[i], now = b->take();
      if (i * b->page < from) {
        src[*pairs] = old;
        dst[*pairs] = now;
        ++*pairs;
      }
      b->put(old);  // others hold it still
      t[i] = now;
    }
  for (int64_t i = held; i < need; ++i) t[i] = b->take();
  b->held[seq] = (int32_t)std::max<int64_t>(held, need);
  return OK;
}

exl3_verdict exl3p_book_fork(exl3p_book *b, int32_t src, int32_t dst, int32_t keys) {
  if (b == nullptr) return refuse(EXL3_FAILED, "PagedBook: a missing argument");
  if (src < 0 || src >= b->seqs || dst < 0 || dst >= b->seqs || src == dst)
    return refuse(EXL3_UNSUPPORTED, "PagedBook: no such sequence");
  if (b->held[dst] != 0) return refuse(EXL3_UNSUPPORTED, "PagedBook: the fork holds pages already");
  if (keys < 0 || b->pages_of(keys) > b->held[src])
    return refuse(EXL3_UNSUPPORTED, "PagedBook: more keys than the sequence holds");
  const int32_t n = (int32_t)b->pages_of(keys);
  const int32_t *from = b->row(src);
  int32_t *to = b->row(dst);
  for (int32_t i = 0; i < n; ++i) {
    to[i] = from[i];
    ++b->refs[from[i]];
  }
  b->held[dst] = n;
  return OK;
}

exl3_verdict exl3p_book_trim(exl3p_book *b, int32_t seq, int32_t keys) {
  if (b == nullptr) return refuse(EXL3_FAILED, "PagedBook: a missing argument");
  if (seq < 0 || seq >= b->seqs) return refuse(EXL3_UNSUPPORTED, "PagedBook: no such sequence");
  if (keys < 0) return refuse(EXL3_UNSUPPORTED, "PagedBook: keys out of order");
  int32_t *t = b->row(seq);
  while (b->held[seq] > b->pages_of(keys)) {
    int32_t &last = t[--b->held[seq]];
    b->put(last);
    last = -1;
  }
  return OK;
}

exl3_verdict exl3p_book_compact(exl3p_book *b, int32_t *src, int32_t *dst, int32_t room,
                                int32_t *pairs) {
  if (b == nullptr || pairs == nullptr || room < 0 ||
      (room > 0 && (src == nullptr || dst == nullptr)))
    return refuse(EXL3_FAILED, "PagedBook: a missing argument");
  *pairs = 0;
  // the highest page in use goes to the lowest free one while that lies below
  // it: no page is both read and written
  std::vector<int32_t> to;
  try {
    to.assign(b->refs.size(), -1);
  } catch (...) {
    return refuse(EXL3_FAILED, "PagedBook: out of host memory");
  }
  int32_t high = (int32_t)b->refs.size() - 1;
  int32_t low = 0;
  while (*pairs < room) {
    while (high >= 0 && b->refs[high] == 0) --high;
    while (low < high && b->refs[low] != 0) ++low;
    if (low >= high) break;
    b->refs[low] = b->refs[high];
    b->refs[high] = 0;
    to[high] = low;
    src[*pairs] = high;
    dst[*pairs] = low;
    ++*pairs;
  }
  if (*pairs == 0) return OK;
  for (int32_t s = 0; s < b->seqs; ++s)
    for (int32_t i = 0; i < b->held[s]; ++i) {
      int32_t &p = b->row(s)[i];
      if (to[p] >= 0) p = to[p];
    }
  // the free pages again, without allocating: as many as before, so the heap's
  // own memory holds them
  while (!b->free.empty()) b->free.pop();
  for (size_t p = 0; p < b->refs.size(); ++p)
    if (b->refs[p] == 0) b->free.push((int32_t)p);
  return OK;
}

const int32_t *exl3p_book_table(const exl3p_book *b) { return b ? b->table.data() : nullptr; }

int32_t exl3p_book_free_pages(const exl3p_book *b) { return b ? (int32_t)b->free.size() : -1; }

int32_t exl3p_book_held(const exl3p_book *b, int32_t seq) {
  return b && seq >= 0 && seq < b->seqs ? b->held[seq] : -1;
}

int32_t exl3p_book_shared(const exl3p_book *b, int32_t page) {
  return b && page >= 0 && (size_t)page < b->refs.size() ? b->refs[page] : -1;
}

}  // extern "C"
