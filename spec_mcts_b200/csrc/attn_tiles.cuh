// Which tiles of keys two tiles of queries of prompt attention go through, and what each of them sees of a tile (attn_tc.cuh): whole numbers alone, which a host compiles too.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define Q40_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define Q40_HOST_DEVICE inline
#endif

namespace q40 {
namespace window {
namespace tc {

constexpr int BQ = 128, BK = 128;            // queries of a tile, keys of a tile

Q40_HOST_DEVICE int larger(int a, int b) { return a > b ? a : b; }
Q40_HOST_DEVICE int smaller(int a, int b) { return a < b ? a : b; }

// Which tiles of keys (by number: keys BK t ..) a tile of queries sees some keys of, and all of them.  (Comparisons of numbers that are made once: the
// thread that issues MMAs asks for every tile, and a few hundred cycles of it were a tenth of the time)
struct Sees {
  int last, from, sinks, all_last, all_from, all_sinks;
  // queries at positions first .. end, none if end < first
  Q40_HOST_DEVICE Sees(int first, int end, int window, int n_sinks) {
    last = end >= first ? end / BK : -1;
    from = first - window + 1 > 0 ? (first - window + 1) / BK : 0;
    sinks = (n_sinks + BK - 1) / BK;
    all_last = (first + 1) / BK - 1;
    all_from = end - window + 1 > 0 ? (end - window + BK) / BK : 0;
    all_sinks = n_sinks / BK;
  }
  Q40_HOST_DEVICE bool some(int t) const { return t <= last && (t >= from || t < sinks); }
  Q40_HOST_DEVICE bool all(int t) const { return t <= all_last && (t >= all_from || t < all_sinks); }
  Q40_HOST_DEVICE bool part(int t) const { return some(t) && !all(t); }
};

// The tiles of keys that a CTA goes through, tile(0) to tile(n - 1): those that one of its queries sees, or a split's share of them
struct Tiles {
  int p_first, p_last;               // positions of the CTA's first and last query
  int t_first, t_from, j0, n;
  // `rows` queries from row0 on
  template <class A>
  Q40_HOST_DEVICE Tiles(const A& a, int row0, int rows, int split) {
    p_first = a.offset + row0;
    p_last = (p_first + rows < a.offset + a.S ? p_first + rows : a.offset + a.S) - 1;
    const int from = p_first - a.window + 1 > 0 ? p_first - a.window + 1 : 0, first = a.sinks < from ? a.sinks : from;
    t_first = (first + BK - 1) / BK;
    t_from = from / BK > t_first ? from / BK : t_first;
    const int all = t_first + p_last / BK + 1 - t_from;
    j0 = (int)((int64_t)all * split / a.splits);
    n = (int)((int64_t)all * (split + 1) / a.splits) - j0;
  }
  Q40_HOST_DEVICE int tile(int j) const { return j + j0 < t_first ? j + j0 : j + j0 - t_first + t_from; }
  // `count` queries from the first-th on
  template <class A>
  Q40_HOST_DEVICE Sees sees(int first, int count, const A& a) const {
    const int end = p_first + first + count - 1;
    return Sees(p_first + first, end < p_last ? end : p_last, a.window, a.sinks);
  }
};

// A row of documents or of a prefix sees keys from `start` on, where its document begins, up to `last`: its own position, or the last of the prefix, which
// is further on.  A row of no document: start is its position, and last one less, or -2 in front of the documents
struct Span { int start, last; };

// The span of a row, documents(k) being where document k begins
template <class A, class D>
Q40_HOST_DEVICE Span span_in(const A& a, int row, D documents) {
  if (documents(0) > row) return {row, -2};
  int k = 0, above = a.n_documents + 1;                // the last that begins at the row or in front of it
  while (above - k > 1) {
    const int mid = (k + above) >> 1;
    if (documents(mid) <= row) k = mid;
    else above = mid;
  }
  if (k == a.n_documents) return {row, row - 1};
  const int start = larger(documents(k), 0), end = smaller(documents(k + 1), a.S);
  const int prefix = smaller(larger(a.prefixes ? a.prefixes[k] : a.prefix, 0), end - start);
  return {start, larger(row, start + prefix - 1)};
}
// ... where all rows are one document
template <class A>
Q40_HOST_DEVICE Span span_of(const A& a, int row) {
  const int p = a.offset + row;
  return {0, larger(p, a.prefix - 1)};
}

// Sees and Tiles for these.  From row to row neither the first key of a window nor `last` falls, so that the first and the last row of a tile tell
struct SpanSees {
  int last, from, sink0, sinks, all_last, all_from, all_sink0, all_sinks;
  // queries at positions p0 .. p1, none if p1 < p0
  Q40_HOST_DEVICE SpanSees(int p0, Span s0, int p1, Span s1, int window, int n_sinks) {
    const int lo0 = larger(s0.start, p0 - window + 1), lo1 = larger(s1.start, p1 - window + 1);
    const bool same = s0.start == s1.start && s0.last >= p0 && s1.last >= p1;
    last = p1 >= p0 ? larger(s1.last, 0) / BK : -1;
    from = lo0 / BK;
    sink0 = s0.start / BK;
    sinks = n_sinks > 0 ? (s0.start + n_sinks - 1) / BK + 1 : 0;
    all_last = same ? (s0.last + 1) / BK - 1 : -1;
    all_from = lo1 > 0 ? (lo1 - 1) / BK + 1 : 0;
    all_sink0 = s0.start > 0 ? (s0.start - 1) / BK + 1 : 0;
    all_sinks = (s0.start + n_sinks) / BK;
  }
  Q40_HOST_DEVICE bool some(int t) const { return t <= last && (t >= from || (t >= sink0 && t < sinks)); }
  Q40_HOST_DEVICE bool all(int t) const { return t <= all_last && (t >= all_from || (t >= all_sink0 && t < all_sinks)); }
  Q40_HOST_DEVICE bool part(int t) const { return some(t) && !all(t); }
};

struct SpanTiles {
  int p_first, p_last;
  int t_sink, t_first, t_from, j0, n;
  bool backwards;                    // scores fall with distance: the largest come first, and no step that follows scales what is there
  // Two tiles of queries from row0 on, the first and the last row of each of which have these spans.  Where the first tile lies in front of all documents, keys begin with what
  // the second one's first row sees.  So one of them goes through each tile of keys, also of documents that do not rise (a row's span ends with the row or behind it, the next
  // one's begins with it or in front), and waits for its copies
  template <class A>
  Q40_HOST_DEVICE SpanTiles(const A& a, int row0, int split, const Span (&at)[4], bool from_the_end) {
    backwards = from_the_end;
    p_first = a.offset + row0;
    p_last = smaller(p_first + 2 * BQ, a.offset + a.S) - 1;
    const bool front = at[1].last == -2, behind = at[0].start == p_first && at[0].last == p_first - 1;           // (behind: so are all rows, and see nothing)
    const int start = front ? at[2].start : at[0].start, from = larger(start, (front ? p_first + BQ : p_first) - a.window + 1), sink_end = smaller(start + a.sinks, from);
    t_sink = start / BK;
    t_first = sink_end > start ? (sink_end - 1) / BK + 1 - t_sink : 0;
    t_from = larger(from / BK, t_sink + t_first);
    const int all = behind || at[3].last < 0 ? 0 : larger(t_first + at[3].last / BK + 1 - t_from, 0);
    j0 = (int)((int64_t)all * split / a.splits);
    n = (int)((int64_t)all * (split + 1) / a.splits) - j0;
  }
  Q40_HOST_DEVICE int tile(int j) const {
    const int at = j0 + (backwards ? n - 1 - j : j);
    return at < t_first ? t_sink + at : at - t_first + t_from;
  }
};

// The rows of a block of two tiles of queries whose spans tell of all of it: the first and the last row of each, the block having n rows
Q40_HOST_DEVICE int edge_row(int e, int n) { return smaller(e == 0 ? 0 : e == 1 ? BQ - 1 : e == 2 ? BQ : n - 1, n - 1); }
// ... and, these being at[0 .. 3], what the block goes through and what each tile of queries sees
struct SpanPlaces {
  SpanTiles tiles;
  SpanSees sees[2];
  template <class A>
  Q40_HOST_DEVICE SpanPlaces(const A& a, int row0, int split, const Span (&at)[4], bool from_the_end)
      : tiles(a, row0, split, at, from_the_end),
        sees{SpanSees(a.offset + row0, at[0], a.offset + row0 + smaller(BQ, smaller(2 * BQ, a.S - row0)) - 1, at[1], a.window, a.sinks),
             SpanSees(a.offset + row0 + BQ, at[2], a.offset + row0 + smaller(2 * BQ, a.S - row0) - 1, at[3], a.window, a.sinks)} {}
};

}  // namespace tc
}  // namespace window
}  // namespace q40
