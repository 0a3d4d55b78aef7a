"""Where the keys and scales of a cache with shared scales lie (csrc/kv_index.h), as a
host program under the sanitizers runs it: blocks of every size, pages through a table
and one a sequence, a page that its last block runs past."""
import pytest

from tests.test_tree_plan import program

TABLE = [[3, -1, 0], [2147483647, 4, 1]]


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    return program(tmp_path_factory, "blocks", """
struct Cache { int pages; int page_shift; int scale_shift; int64_t capacity; int64_t sp, sh, ss, scp, sch, scs;
               const int32_t* table; int64_t table_stride; };
int main(int, char** v) {
  const std::vector<int32_t> table = {3, -1, 0, 2147483647, 4, 1}, ctx = {5, 0};
  const int paged = atoi(v[1]), shift = atoi(v[2]), scale = atoi(v[3]), size = atoi(v[4]);
  Cache c{5, shift, scale, paged ? 3ll << shift : size, 1ll << 40, 70000, 64, 1ll << 33, 5000, 3,
          paged ? table.data() : nullptr, 3};
  for (int64_t b = 0; b < 2; ++b)
    for (int64_t n = 0; n < c.capacity + 2; ++n) {
      const auto s = frisk::kv::slot_of(c, b, n);
      const int entry = frisk::tree::entry_of(c, ctx.data(), b, (int)n);
      const auto p = frisk::tree::place_of(c, 1, b, 2, (int)n, (int)c.capacity, entry);
      printf("%lld %lld %lld %lld %d %lld %lld\\n", (long long)b, (long long)n, (long long)s.elem, (long long)s.scale,
             (int)p.there, (long long)p.row, (long long)p.scale);
    }
}""")


@pytest.mark.parametrize("paged,shift,scale,size", [
    (1, 8, 8, 0), (1, 8, 0, 0), (1, 6, 5, 0), (1, 4, 4, 0), (1, 3, 1, 0),
    (0, 0, 5, 100), (0, 0, 8, 300), (0, 0, 8, 7), (0, 0, 3, 64), (0, 0, 0, 33)])
def test_scales_of_blocks(index, paged, shift, scale, size):
    page, cap = (1 << shift, 3 << shift) if paged else (size, size)
    seen = 0
    for b, n, elem, at, there, row, head_at in index(paged, shift, scale, size):
        pg, slot = (TABLE[b][n // page], n % page) if paged and n < cap else (b, n)
        if n < cap and 0 <= pg < 5:
            assert (elem, at) == ((pg << 40) + slot * 64, (pg << 33) + slot // (1 << scale) * 3)
            assert (there, row, head_at) == (1, elem + 2 * 70000, at + 2 * 5000)
            seen += 1
        else:
            assert (elem, at) == (-1, -1) and (there, row, head_at) == (0, 2 * 70000, 2 * 5000)
    assert seen == (4 * page if paged else 2 * size)
