// Which states the tokens of a sliding window read, which rows read a state, and how a call's walks over both are cut into parts: whole-number
// arithmetic alone, for the kernels, for the host that launches them, and for a compiler that knows nothing of CUDA.
//
// Token t of a sequence stands at place offset + t and reads the states [place - before, place + after] and, of the first `sinks`, those up to
// place + after.  Offsets and reaches are any 64-bit numbers: their sums are formed without overflow and brought to +-2^40, beyond which they
// say no more (tokens and states are fewer than 2^30).  P: a call's parameters (AttnParams).
#pragma once

#ifdef __CUDACC__
#define MVR_EVERYWHERE __host__ __device__ __forceinline__
#else
#define MVR_EVERYWHERE inline
#endif

namespace mvr {

MVR_EVERYWHERE long long smaller(long long a, long long b) { return a < b ? a : b; }
MVR_EVERYWHERE long long larger(long long a, long long b) { return a > b ? a : b; }
MVR_EVERYWHERE long long parts_of(long long a, long long b) { return (a + b - 1) / b; }  // a >= 0: how many of b hold a

// ---- a token's states ---------------------------------------------------------------------------------
// Token t reads the states [lo + t, hi + t) (and first ones before hi + t).
struct Places {
  long long lo, hi;
};
MVR_EVERYWHERE long long near_sum(long long a, long long b) {
  const long long sum = (long long)((unsigned long long)a + (unsigned long long)b);
  const long long most = 1ll << 40;
  if (((a ^ sum) & (b ^ sum)) < 0) return a < 0 ? -most : most;  // beyond 64 bits
  return larger(-most, smaller(sum, most));
}
MVR_EVERYWHERE Places places_from(long long offset, long long before, long long after) {  // (before and after are not negative)
  return {near_sum(offset, -before), near_sum(offset, after) + 1};
}

// The states [lo, hi) and [0, sink).
struct Span {
  int lo, hi, sink;
};
// Of the tokens `first` to `last`, together, among `end` states: neighbouring tokens leave no gap between their windows.
template <typename P>
MVR_EVERYWHERE Span span_of(const P& p, const Places& at, int first, int last, int end) {
  Span s;
  s.hi = (int)larger(0, smaller(at.hi + last, end));
  s.lo = (int)larger(0, smaller(at.lo + first, s.hi));
  s.sink = p.sinks < s.hi ? p.sinks : s.hi;
  return s;
}
MVR_EVERYWHERE unsigned bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }
// Which of the states j to j + 31 lie in it.
MVR_EVERYWHERE unsigned span_bits(const Span& s, int j) {
  return (bits_below(s.hi - j) & ~bits_below(s.lo - j)) | bits_below(s.sink - j);
}
// The tiles of STEP states that hold a span: those of the first states, then those of the window from its own beginning on.
template <int STEP>
struct SpanTiles {
  int sinks, from, count;
  MVR_EVERYWHERE SpanTiles(const Span& s) {
    sinks = (s.sink + STEP - 1) / STEP;
    from = s.lo > sinks * STEP ? s.lo : sinks * STEP;  // (what lies before is in the first ones' tiles)
    count = sinks + (s.hi > from ? s.hi - from + STEP - 1 : 0) / STEP;
  }
  MVR_EVERYWHERE int first(int i) const { return i < sinks ? i * STEP : from + (i - sinks) * STEP; }
};

// ---- a state's rows -----------------------------------------------------------------------------------
// A CTA takes a tile of states and a part of the rows whose windows reach it.  All tokens may read the first tiles, so those are cut
// into more parts, which come first: sink_parts of each of the sink_tiles of an image, then row_splits of each of the others.
struct StateTile {
  int n, tile, part;
  bool sink;
};
template <typename P>
MVR_EVERYWHERE StateTile state_tile(const P& p, int block, int state_tiles) {
  const int leading = p.N * p.sink_tiles * p.sink_parts;
  StateTile s;
  s.sink = block < leading;
  const int at = block - (s.sink ? 0 : leading), parts = s.sink ? p.sink_parts : p.row_splits;
  const int number = at / parts, tiles = s.sink ? p.sink_tiles : state_tiles - p.sink_tiles;
  s.part = at - number * parts;
  s.n = number / tiles;
  s.tile = number - s.n * tiles + (s.sink ? 0 : p.sink_tiles);
  return s;
}
// Rows of a key head that read state j: [lo, hi).
template <typename P>
MVR_EVERYWHERE void rows_of_state(const P& p, const Places& at, int j, int& lo, int& hi) {
  lo = (int)larger(0, smaller(j + 1 - at.hi, p.T)) * p.G;
  hi = (j < p.sinks ? p.T : (int)larger(0, smaller(j + 1 - at.lo, p.T))) * p.G;
}
// The part's tiles of `step` rows for the states from j0 on, `size` of them, among `end`: the first row, how many tiles, and behind which row
// none reads any of the states: what such a row holds may not come near their sums.
struct TileRows {
  int first, count, end;
};
template <typename P>
MVR_EVERYWHERE TileRows rows_of_states(const P& p, const StateTile& s, const Places& at, int j0, int size, int end, int step) {
  int lo, hi, unused;
  rows_of_state(p, at, j0, lo, hi);
  if (j0 >= p.sinks) rows_of_state(p, at, (int)smaller(j0 + size, end) - 1, unused, hi);
  const int all = (hi > lo ? hi - lo + step - 1 : 0) / step;
  const int per = s.sink ? (all + p.sink_parts - 1) / p.sink_parts : p.row_tiles_per;
  const int left = all - s.part * per;
  return {lo + s.part * per * step, left < 0 ? 0 : left < per ? left : per, hi};
}
// Where a state's sums of a part go: parts of the first tiles lie before those of the others, each without the other's states.
struct PartPlace {
  bool parts;
  long long at;
};
template <typename P>
MVR_EVERYWHERE PartPlace part_place(const P& p, const StateTile& s, int j, int hk, int tile) {
  const long long lead = smaller(p.L, (long long)p.sink_tiles * tile), states = s.sink ? lead : p.L - lead, row = (long long)p.Hk * p.D;
  PartPlace r;
  r.parts = (s.sink ? p.sink_parts : p.row_splits) > 1;
  r.at = (((long long)s.part * p.N + s.n) * states + (s.sink ? j : j - lead)) * row + (long long)hk * p.D;
  if (!s.sink && p.sink_parts > 1) r.at += p.sink_parts * (p.N * lead * row);
  return r;
}

// ---- how walks are cut (host) ---------------------------------------------------------------------------
// Sizes of a call, reaches cut to what exceeds any size.
struct WindowSizes {
  long long T, L, G, before, after, sinks;
  // the most states that `tokens` neighbouring tokens read in their windows
  long long reach(long long tokens) const { return smaller(L, tokens + before + after); }
  // the most tiles of `size` states of a span of `rows` rows
  long long span_tiles(long long rows, long long size) const {
    const long long tokens = smaller(T, parts_of(rows, G) + 1);
    return larger(1, smaller(parts_of(L, size), parts_of(reach(tokens), size) + 1 + parts_of(sinks, size)));
  }
  // the most rows that read one of `states` neighbouring states beyond the first ones
  long long rows_reached(long long states) const { return smaller(T, states + before + after) * G; }
  // tiles of `step` rows of one of `parts` parts of the rows of `states` states
  int row_tiles(long long states, long long step, long long parts) const {
    return (int)larger(1, parts_of(smaller(parts_of(T * G, step), parts_of(rows_reached(states), step) + 1), parts));
  }
  // parts, as long, into which the rows of the first states are cut
  int sink_parts(long long step, int row_tiles_per) const { return (int)larger(1, smaller(64, parts_of(parts_of(T * G, step), row_tiles_per))); }
};
inline WindowSizes window_sizes(long long T, long long L, long long G, long long before, long long after, long long sinks) {
  const long long most = 1ll << 31;
  return {T, L, G, smaller(before, most), smaller(after, most), smaller(sinks, L)};
}

}  // namespace mvr
