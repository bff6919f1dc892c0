// Host program of test_window_geometry.py: replays the window kernels' tile lists and the
// masks' rule on the CPU, from the kernels' own headers.  Each line of standard input is
// "L S left right sinks bm bn kg splits"; each line of output "ok" or what is wrong.
//
// A row's visible keys, by the definition, must lie in exactly one tile of its block's
// list, in a round and key group that its wave computes; the tiles must begin at keys of
// the sequence, and the splits' shares must cover the list once.
#include <stdio.h>

#include <vector>

#include "../cpu-attention_amd/csrc/ca_window.h"

using namespace ca;

static const char* check(WindowParams p, int bm, int bn, int kg, int splits) {
  const int L = (int)p.seq_q, S = (int)p.seq_k;
  for (int q0 = 0; q0 < L; q0 += bm) {
    const WinTiles w = win_tiles(p, q0, bm, bn);
    if (w.n < 0 || w.n > win_most_tiles(p, bm, bn)) return "tile count";
    std::vector<int> covered(S, 0), tile_of(S, -1);
    for (int t = 0; t < w.n; ++t) {
      const int k0 = win_key0(w, t, bn);
      if (k0 < 0 || k0 >= S) return "a tile begins outside the sequence";
      for (int j = k0; j < k0 + bn && j < S; ++j) {
        ++covered[j];
        tile_of[j] = t;
      }
    }
    for (int r0 = q0; r0 < q0 + bm; r0 += 32) {
      std::vector<int> done(w.n, 0);
      for (int sp = 0; sp < splits; ++sp)
        for (int g = 0; g < kg; ++g) {
          const WinRounds r = win_rounds(p, w, bn, r0, sp, splits, kg, g);
          if (r.nkt_w > r.nkt || r.nkt < 0) return "rounds";
          const int share = (w.n + splits - 1) / splits;
          for (int t = 0; t < r.nkt_w; ++t) {
            const int i = r.t0 + t * kg + g;
            if (i >= w.n || i >= r.t0 + share) return "a round past the share";
            ++done[i];
          }
        }
      for (int t = 0; t < w.n; ++t)
        if (done[t] > 1) return "a tile computed twice";
      for (int i = r0; i < r0 + 32 && i < L; ++i) {
        const long pos = (long)i + S - L;
        for (int j = 0; j < S; ++j) {
          const bool seen = j <= pos + p.right && (j >= pos - p.left || j < p.sinks);
          if (seen != win_sees(p, (int)pos, j)) return "the rule";
          if (seen && covered[j] != 1) return "a visible key not in one tile";
          if (seen && !done[tile_of[j]]) return "a visible key's tile not computed";
        }
      }
    }
  }
  return "ok";
}

int main() {
  int L, S, left, right, sinks, bm, bn, kg, splits;
  while (scanf("%d %d %d %d %d %d %d %d %d", &L, &S, &left, &right, &sinks, &bm, &bn, &kg, &splits) == 9) {
    WindowParams p{};
    p.batch = p.heads = 1;
    p.seq_q = L;
    p.seq_k = S;
    p.left = left;
    p.right = right;
    p.sinks = sinks;
    printf("%s\n", check(p, bm, bn, kg, splits));
  }
  return 0;
}
