// Integer side of the paged key-value cache, shared by the kernels and the host (the CPU unit tests call the same code
// through the host entry points): which keys the one new token of a sequence sees, the 16-key steps that cover them, and
// the rules for page-table entries.
//
// A cache tensor holds num_pages pages of page_size rows; key j of sequence b is row j % page_size of page
// block_table[b][j / page_size]. An entry outside [0, num_pages) holds no keys: the positions it stands for are not
// visible (a program that keeps a window gives the pages between the sinks and the window back and writes -1 there).
#pragma once
#include <stdint.h>

#include "attn_index.h"

namespace b200fa {

constexpr int kPagedStep = 16;  // keys per step of the decoding kernel

// The new token is the last of its sequence (row len - 1), so it sees keys [lo, len) and, in front of them, the first
// `sink`. The steps that hold visible keys are numbered without the gap between the sinks and the window: step v is
// v for v < sink_steps and v + gap behind them.
struct PagedRange {
  int len, lo, sink;
  int sink_steps, gap, steps;
  B200FA_HD bool sees(int key) const { return key < len && (key >= lo || key < sink); }
  B200FA_HD int step_of(int v) const { return v < sink_steps ? v : v + gap; }
};

// `capacity` = keys that the table has entries for; lengths outside [0, capacity] are cut to it.
B200FA_HD PagedRange paged_range(int length, int capacity, int left, int sink) {
  PagedRange r;
  r.len = imin(imax(length, 0), capacity);
  r.lo = left < 0 ? 0 : imax(0, r.len - 1 - left);
  r.sink = imin(sink, r.lo);
  r.sink_steps = ceil_div(r.sink, kPagedStep);
  const int first = imax(r.lo / kPagedStep, r.sink_steps), last = (r.len + kPagedStep - 1) / kPagedStep;
  r.gap = first - r.sink_steps;
  r.steps = r.sink_steps + imax(last - first, 0);
  return r;
}

}  // namespace b200fa
