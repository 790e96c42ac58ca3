// Index arithmetic of the paged key/value cache, in plain C++ so that it is tested on the CPU as well: which page a token is
// in, which rows of a page an append writes, and what a wrong table, length or position is turned into.  Everything that the
// kernels read or write of the cache goes through these functions.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define DSB_HD __host__ __device__ __forceinline__
#else
#define DSB_HD inline
#endif

namespace dsb {

// Page of a sequence's tokens [j * T, (j + 1) * T), or -1 where the table ends or names no page of the pool.
DSB_HD int kv_page(const int32_t* table_row, int width, int n_pages, int j) {
  if (j < 0 || j >= width) return -1;
  const int page = table_row[j];
  return page >= 0 && page < n_pages ? page : -1;
}

// Length of a sequence as the kernels use it: never negative, never past its table.
DSB_HD int kv_length(int len, int64_t capacity) {
  if (len < 0) return 0;
  return len > capacity ? static_cast<int>(capacity) : len;
}
DSB_HD bool kv_length_ok(int len, int64_t capacity) { return len >= 0 && len <= capacity; }

// Keys that query i of Sq sees of a sequence of `len` keys: all, or (causal) those up to its own position len - Sq + i.
DSB_HD int kv_visible(int len, int Sq, int i, int causal) {
  if (!causal) return len;
  const int n = len - Sq + i + 1;
  return n < 0 ? 0 : n;
}

// Rows that an append of `count` tokens from position `start` on puts into its j-th page (T tokens a page).
struct KvSpan {
  int index;  // of the page in the sequence's table
  int slot;   // first slot written
  int row;    // first of the appended rows that goes there
  int rows;   // how many (0: this page is not touched)
};
DSB_HD KvSpan kv_span(int start, int count, int T, int j) {
  KvSpan s;
  s.index = start / T + j;
  s.slot = j == 0 ? start % T : 0;
  s.row = j == 0 ? 0 : j * T - start % T;
  const int left = count - s.row;
  const int room = T - s.slot;
  s.rows = left <= 0 ? 0 : (left < room ? left : room);
  return s;
}
// Pages that n rows can touch, wherever they start.
DSB_HD int kv_span_pages(int n, int T) { return (n + T - 2) / T + 1; }

// Whether an append of a sequence may run: a position and a count inside its table.
DSB_HD bool kv_append_ok(int start, int count, int n, int64_t capacity) {
  return start >= 0 && count >= 0 && count <= n && static_cast<int64_t>(start) + count <= capacity;
}

// The least e in [-64, 64] with |x| <= 448 * 2^e, from the bits of a finite |x|: 448 = 1.75 * 2^8.
DSB_HD int kv_exponent(uint32_t abs_bits) {
  const int e = static_cast<int>(abs_bits >> 23) - 127 - 8 + ((abs_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -64 ? -64 : (e > 64 ? 64 : e);
}

// A block's exponent as the kernels use it: what a caller has put there outside -64..64 counts as the nearer end.
DSB_HD int kv_held_exponent(int e) { return e < -64 ? -64 : (e > 64 ? 64 : e); }

// Whether a stream's record of an item that goes on in the `more` streams behind it names an item and streams that there are; the combine
// pass makes addresses of it.
DSB_HD bool kv_cut_ok(int pair, int h, int more, int slot, int stream, int pairs, int heads, int n_streams) {
  return pair >= 0 && pair < pairs && h >= 0 && h < heads && more > 0 && more < n_streams - stream && (slot == 0 || slot == 1);
}

}  // namespace dsb
