// Which of a request's cached tokens a tile of query rows has to look at.
#pragma once

namespace qs {

// Tokens [lo, hi).  An empty span is [0, 0): rounded to whole steps of tokens it has none, so nothing is
// looked up for it in a block table.
struct Span {
  int lo, hi;
};

// Tokens that some of the rows see, which stand at pos_min .. pos_max of a request (any: it has a context).
// A table row has room for `reach` tokens, and hi never passes that; a window may end before it begins
// there, where the context is longer than the table.
constexpr Span span_of(int pos_min, int pos_max, int window, int reach, bool any) {
  Span s{window > 0 && pos_min >= window ? pos_min - window + 1 : 0, pos_max < reach ? pos_max + 1 : reach};
  if (!any || s.hi <= s.lo) s = Span{0, 0};
  return s;
}

}  // namespace qs
