// The key lists of windowed prefill items.
#pragma once

#include "paged_attention.hpp"

namespace mvllm {

// The key list of an item whose first query stands at position p0 (paged_attention.hpp): entry v
// at position v for v < front, v + gap from there on, front a multiple of `align`. [hole, seen) are
// the entries that no query of the item sees: none with align 1; with align a run of `align`
// keys always holds a key that is seen, so the page of such a run is the sequence's own still.
struct WindowList {
  int front, gap, hole, seen;
};
template <int align>
__device__ __forceinline__ WindowList window_list(const PagedParams& p, int p0) {
  WindowList w;
  const int lo = max(p0 - p.window + 1, 0);  // the first key of the first query's window
  w.front = min(p.sinks, lo);
  w.front = (w.front + align - 1) / align * align;
  w.gap = max(lo / align * align - w.front, 0);
  w.seen = lo - w.gap;
  w.hole = min(p.sinks, w.seen);
  return w;
}
__device__ __forceinline__ int list_position(const WindowList& w, int v) {
  return v < w.front ? v : v + w.gap;
}

}  // namespace mvllm
