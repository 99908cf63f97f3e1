// The launches of causal attention (train_attention.h): every tile of rows once, last
// ones first within a head, and no workgroups for tiles that there are not.
#include "train_attention.h"

#include <cstdio>
#include <vector>

using namespace mfh;
using namespace mfh::attend;

static int Fail(const char *what, const TrainAttention &a) {
  std::printf("%s: batch %d heads %d over %d queries %d keys %d dim %d\n", what, a.batch, a.heads,
              a.kv_heads, a.q_len, a.k_len, a.dim);
  return 1;
}

int main() {
  for (int batch : {1, 3, 64, 1024})
    for (int kv : {1, 3})
      for (int group : {1, 2, 3, 8, 100, 128})
        for (int q_len : {1, 2, 9, 63, 64, 65, 129, 300, 1021})
          for (int k_len : {1, 64, 2000})
            for (int dim : {32, 128}) {
              TrainAttention a;
              a.batch = batch;
              a.kv_heads = kv;
              a.group = group;
              a.heads = kv * group;
              a.q_len = q_len;
              a.k_len = k_len;
              a.dim = dim;
              a.dtype = DT_BF16;
              a.causal = true;
              Args s = ArgsOf(a, false);
              const int tiles = s.tiles, lines = (s.lines + 7) / 8 * 8;
              const std::int64_t groups = GroupsOf(&s);
              if (s.splits > 1)
                continue;  // in order
              if (s.down < 1)
                return Fail("no order", a);
              // Each head's last run may be short of a tile.
              const int places = PlacesDown(tiles, s.down), each = (tiles + group - 1) / group;
              if (places >= tiles + each)
                return Fail("workgroups without a tile", a);
              if (groups > static_cast<std::int64_t>(lines) * (tiles + each - 1))
                return Fail("a launch too large", a);
              std::vector<int> when(tiles, -1);
              for (int at = 0; at < places; ++at) {
                const int tile = TileDown(at, tiles, s.down);
                if (tile < 0)
                  return Fail("a tile below the first", a);
                if (tile >= tiles)
                  continue;
                if (when[tile] >= 0)
                  return Fail("a tile twice", a);
                when[tile] = at;
              }
              const int run = (tiles + s.down - 1) / s.down;
              for (int tile = 0; tile < tiles; ++tile) {
                if (when[tile] < 0)
                  return Fail("a tile left out", a);
                if (tile % run && when[tile] > when[tile - 1])
                  return Fail("an early tile first", a);
              }
            }
  std::printf("attention order ok\n");
  return 0;
}
