// Every block-table column that attention over the 4-bit cache looks up lies in the table, and every
// token that a row sees lies in a step that is taken.
//
// Walks positions, windows and table widths, and for each tile takes the kernels' steps (of 32 or 64
// tokens, split into parts or not) and their lookups, one for 16 tokens, of the tokens below the
// span's end.  Exit status 0 iff no lookup is out of range and no seen token is left out.
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "../mrun-pub_amd/csrc/qs_span.h"

static long looked = 0, bad = 0, lost = 0;

static void walk(int pos_min, int pos_max, int window, int64_t width, int shift, int step, int parts) {
  const int64_t room = width << shift;
  const int reach = (int)(room < (1 << 30) ? room : 1 << 30);
  const qs::Span s = qs::span_of(pos_min, pos_max, window, reach, true);
  const int first = s.lo / step, steps = (s.hi + step - 1) / step - first;
  for (int part = 0; part < parts; ++part) {
    const int s0 = first + (int)((int64_t)steps * part / parts), s1 = first + (int)((int64_t)steps * (part + 1) / parts);
    for (int i = s0; i < s1; ++i)
      for (int64_t t = (int64_t)i * step; t < (int64_t)(i + 1) * step; t += 16) {
        if (t >= s.hi) continue;
        ++looked;
        if (t < 0 || (t >> shift) >= width) ++bad;
      }
  }
  for (int pos = pos_min; pos <= pos_max; ++pos)
    for (int64_t t = window > 0 && pos >= window ? pos - window + 1 : 0; t <= pos; ++t) {
      if (t >= reach) break;
      if (t < s.lo || t >= s.hi || t / step < first || t / step >= first + steps) ++lost;
      if (t > 300 && t + 300 < pos) t = pos - 300;  // the middle of long contexts is like its ends
    }
}

int main() {
  for (int step = 32; step <= 64; step += 32)
    for (int parts = 1; parts <= 3; parts += 2)
      for (int shift = 4; shift <= 8; shift += 2)
        for (int width = 0; width <= 5; ++width) {
          const int reach = width << shift;
          for (int window : {0, 1, 2, 5, 17, 31, 32, 33, 100, 257})
            for (int rows : {1, 2, 5, 33}) {
              for (int pos = -40; pos <= reach + 700; ++pos) walk(pos, pos + rows - 1, window, width, shift, step, parts);
              for (int pos : {1 << 20, (1 << 30) - 40, 1 << 30})
                if (window > 0) walk(pos, pos + rows - 1, window, width, shift, step, parts);
            }
        }
  std::printf("lookups %ld, out of range %ld, seen tokens left out %ld\n", looked, bad, lost);
  return bad || lost || !looked;
}
