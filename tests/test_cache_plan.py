"""How the blocks of attention over a paged cache share out its walk: what the host makes room for is enough for whatever lengths come, up to 2^31 tokens."""
import os
import subprocess

CHECK = r"""
#include <cstdio>
#include <initializer_list>
#include "cache_plan.hpp"
using namespace b200;
typedef unsigned long long u64;
static u64 seed = 1;
static u64 below(u64 n) { seed = seed * 6364136223846793005ull + 1442695040888963407ull; return (seed >> 33) % n; }
int main() {
  int bad = 0;
  for (u64 capacity = 1; capacity <= (1ull << 25); capacity += 1 + capacity / 7)
    for (u64 tiles : {1ull, 2ull, 3ull, 8ull, 61ull, 256ull, 2049ull})
      for (unsigned blocks : {148u, 296u, 592u}) {
        const CachePlan p = cache_plan(tiles, capacity, blocks, 4, 256);
        if (p.single) continue;
        for (int t = 0; t < 8; ++t) {
          // tiles that see all that the table may hold, and fewer of them, of which the last one may be shorter
          const u64 some = t == 0 ? tiles : 1 + below(tiles), length = t < 2 ? capacity : 1 + below(capacity), all = some * length;
          const u64 quota = cache_quota((all + blocks - 1) / blocks, p.least), needed = (all + quota - 1) / quota;
          bool fine = quota <= kCachePart && quota >= p.least && needed <= p.grid;
          // the parts of each tile are blocks of the grid; those that reach the joining together are 256 at most while a part is no longer than `least`
          for (u64 i = 0; i < some; i += 1 + some / 5) {
            const u64 from = i * length, first = from / quota, parts = (from + length - 1) / quota - first + 1;
            fine = fine && first + parts <= p.grid && (quota == kCachePart || parts <= 256);
          }
          if (!fine && bad++ < 5) printf("capacity %llu tiles %llu of %llu blocks %u: least %u grid %llu needed %llu\n", capacity, some, length, blocks, p.least, p.grid, needed);
        }
      }
  printf("%d\n", bad);
  return bad != 0;
}
"""


def test_the_grid_holds_every_walk(tmp_path):
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ocannl_b200", "csrc")
    src, exe = tmp_path / "plan.cpp", str(tmp_path / "plan")
    src.write_text(CHECK)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", root, str(src), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
