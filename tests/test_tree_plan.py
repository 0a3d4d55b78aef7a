"""Host programs over the rules and the indexing of attention over a cache
(csrc/launch_plan.h, csrc/kv_index.h): which kernel a call takes and how its
keys are split, where keys lie (pages that are none, lengths behind the
capacity), which keys a token sees."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "frisk_amd", "csrc")
ROWS, KEYS, TILE4, TILE8 = range(4)


def program(tmp_path_factory, name, body):
    d = tmp_path_factory.mktemp(name)
    src, exe = d / "main.cpp", d / "main"
    src.write_text(f"""#include "{CSRC}/launch_plan.h"
#include "{CSRC}/kv_index.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
{body}""")
    subprocess.run(["g++", "-std=c++17", "-fsanitize=address,undefined", "-fno-sanitize-recover", str(src), "-o",
                    str(exe)], check=True)

    def run(*args):
        out = subprocess.run([str(exe), *(str(a) for a in args)], check=True, capture_output=True, text=True).stdout
        return [[int(x) for x in line.split()] for line in out.strip().split("\n")]
    return run


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    run = program(tmp_path_factory, "plan", """
using namespace frisk::plan;
int main(int, char** v) {
  const auto n = [&](int i) { return (int64_t)atoll(v[1 + i]); };
  const TreePlan p = tree_plan(n(0), n(1), n(2), n(3), n(4), n(5), n(6), n(7), 256);
  printf("%d %d %d %lld\\n", (int)p.kernel, p.splits, p.min_blocks,
         (long long)tree_workspace(p, n(0), n(1), n(2), n(3), n(4)));
}""")
    return lambda batch, heads, kv, tokens, d, bits8, keys, split=1: run(batch, heads, kv, tokens, d, bits8, keys,
                                                                        split)[0]


def test_rule_picks_the_measured_kernels(plan):
    # One token, few drafts, many rows, chunks; head dims without a matrix-core kernel.
    assert plan(8, 32, 8, 1, 128, 0, 8193)[0] == KEYS
    assert plan(8, 32, 8, 16, 128, 1, 8208)[0] == KEYS
    assert plan(8, 32, 8, 24, 128, 0, 8216)[0] == TILE4
    assert plan(8, 32, 8, 64, 128, 0, 8256)[0] == TILE8
    assert plan(2, 32, 8, 512, 128, 0, 32768)[0] == TILE8
    assert plan(2, 32, 8, 512, 64, 1, 8704)[0] == TILE4
    for d in (16, 48, 80, 96, 256):
        assert plan(2, 8, 2, 5, d, 0, 4096)[0] == ROWS
    # The shapes of the GPU tests that are meant for the tiled kernels.
    for bits8 in (0, 1):
        for d, keys in ((32, 624), (64, 816), (128, 816)):
            assert plan(4, 16, 4, 512, d, bits8, keys)[0] == TILE4
        assert plan(8, 16, 4, 512, 128, bits8, 816)[0] == TILE8
    kernel, splits, *_ = plan(8, 32, 8, 64, 128, 0, 4160)
    assert kernel == TILE8 and splits > 1
    kernel, splits, *_ = plan(2, 32, 8, 64, 128, 0, 8256)
    assert kernel == TILE4 and splits > 1


def test_splits_and_workspace(plan):
    for args in ((1, 32, 8, 1, 128, 0, 100000), (1, 8, 8, 1, 64, 1, 5000), (2, 32, 8, 64, 128, 1, 30000),
                 (1, 4, 1, 3, 80, 0, 9000), (64, 32, 8, 1, 128, 0, 2048), (1, 1, 1, 1, 32, 0, 1)):
        kernel, splits, least, ws = plan(*args)
        b, h, kv, t, d, _, keys = args
        assert 1 <= splits <= 64 and splits * least <= max(least, -(-keys // 64))
        assert (ws == 0) == (splits == 1)
        if splits > 1:
            rows = b * kv * -(-t * (h // kv) // 32) * 32 if kernel == KEYS else b * h * t
            assert ws >= rows * splits * (d + 2) * 4
        # Without a workspace there are none.
        assert plan(*args, 0)[1] == 1


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    return program(tmp_path_factory, "index", """
struct Cache { int pages; int page_shift; int64_t capacity; int64_t sp, sh, ss, scp, sch, scs;
               const int32_t* table; int64_t table_stride; };
int main(int, char** v) {
  // Two sequences of 4 pages of 8 keys; pages -1, 7 (of 5) and 2^31 - 1 are none.
  const std::vector<int32_t> table = {3, -1, 7, 0, 2147483647, 1, 4, -2147483647}, ctx = {5, -1};
  const bool paged = atoi(v[1]);
  Cache c{5, 3, paged ? 32 : 20, 1000000000000, 7000, 64, 900, 70, 1, paged ? table.data() : nullptr, 4};
  for (int64_t b = 0; b < 2; ++b)
    for (int64_t n : {-1ll, 0ll, 7ll, 8ll, 15ll, 16ll, 19ll, 20ll, 23ll, 24ll, 31ll, 32ll, 1ll << 40}) {
      const auto s = frisk::kv::slot_of(c, b, n);
      const int entry = frisk::tree::entry_of(c, ctx.data(), b, (int)(n > 1000 ? 1000 : n));
      const auto p = frisk::tree::place_of(c, 2, b, 1, (int)(n < 0 ? 0 : n > 1000 ? 1000 : n), (int)c.capacity, entry);
      printf("%lld %lld %lld %lld %d %lld %lld\\n", (long long)b, (long long)n, (long long)s.elem, (long long)s.scale,
             (int)p.there, (long long)p.row, (long long)p.scale);
    }
}""")


@pytest.mark.parametrize("paged", [0, 1])
def test_keys_outside_the_cache_have_no_place(index, paged):
    table = [[3, -1, 7, 0], [2147483647, 1, 4, -2147483647]]
    cap = 32 if paged else 20
    for b, n, elem, scale, there, row, srow in index(paged):
        page, slot = (table[b][n // 8], n % 8) if paged and 0 <= n < cap else (b, n)
        if 0 <= n < cap and 0 <= page < 5:
            assert (elem, scale) == (page * 10 ** 12 + slot * 64, page * 900 + slot)
            assert (there, row, srow) == (1, 2 * (elem + 7000), scale + 70)
        else:
            assert (elem, scale) == (-1, -1)
            if n >= 0:  # a load goes to the first row of the head, hidden
                assert (there, row, srow) == (0, 2 * 7000, 70)


@pytest.fixture(scope="module")
def masks(tmp_path_factory):
    return program(tmp_path_factory, "masks", """
int main(int, char** v) {
  const int tokens = atoi(v[1]), ctx = atoi(v[2]), causal = atoi(v[3]), words = (tokens + 63) / 64;
  for (int t = 0; t < tokens; ++t) {
    std::vector<uint64_t> w(words);
    for (int j = 0; j < tokens; ++j)
      if ((t * 37 + j * 11 + t * j) % 5 < 2) w[j / 64] |= 1ull << (j % 64);
    for (int n0 = 0; n0 < ctx + tokens; n0 += 64) {
      const int left = ctx + tokens - n0;
      const uint64_t there = left >= 64 ? ~0ull : (1ull << left) - 1;
      const uint64_t s = frisk::tree::seen_bits(causal ? nullptr : w.data(), tokens, t, ctx, n0, there);
      printf("%d %d %lld %lld\\n", t, n0, (long long)(s >> 32), (long long)(s & 0xffffffffu));
    }
  }
}""")


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("tokens,ctx", [(1, 0), (1, 63), (1, 64), (7, 60), (64, 0), (64, 1), (65, 63), (130, 100), (200, 64)])
def test_seen_bits(masks, tokens, ctx, causal):
    for t, n0, hi, lo in masks(tokens, ctx, causal):
        bits = hi << 32 | lo
        for i in range(64):
            n = n0 + i
            j = n - ctx
            want = n < ctx or (j < tokens and (j <= t if causal else (t * 37 + j * 11 + t * j) % 5 < 2))
            assert (bits >> i & 1) == want, (t, n)


def test_sequences_divide_into_splits(tmp_path_factory):
    run = program(tmp_path_factory, "cut", """
int main(int, char**) {
  for (int splits : {1, 2, 3, 7, 64})
    for (int least : {1, 4, 8})
      for (int blocks : {0, 1, 3, 4, 5, 31, 32, 33, 1000}) {
        const int per = frisk::tree::blocks_per_split(splits, least, blocks);
        printf("%d %d %d %d\\n", splits, least, blocks, per);
      }
}""")
    for splits, least, blocks, per in run():
        used = max(1, -(-blocks // per))
        assert per >= least and used <= splits and used * per >= blocks


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("batch,heads,kv,tokens", [
    ((1 << 24) - 1, 1, 1, 1), ((1 << 23) + 1, 1, 1, 1), (1 << 23, 1, 1, 1), (1 << 18, 60, 30, 1), (1 << 19, 31, 31, 1),
    (1 << 22, 3, 3, 1), (255, 65535, 65535, 1), (1, 1, 1, (1 << 24) - 1), (1, 4, 2, 1 << 21)])
def test_every_call_fits_a_launch(plan, batch, heads, kv, tokens, d):
    # Up to 2^24 - 1 query rows are taken: a launch has fewer than 2^32 threads.
    for keys in (1, 100, 5000):
        for bits8 in (0, 1):
            kernel, splits, *_ = plan(batch, heads, kv, tokens, d, bits8, keys)
            tile, threads = {ROWS: (1, 256), KEYS: (32, 256 if d == 128 else 512), TILE4: (128, 256),
                             TILE8: (256, 512)}[kernel]
            units = batch * heads * tokens if kernel == ROWS else batch * kv * -(-tokens * (heads // kv) // tile)
            assert units * splits * threads < 2 ** 32


@pytest.mark.parametrize("batch,heads,kv,tokens,d,bits8,keys,least,most", [
    (1, 32, 8, 1, 128, 0, 32768, 12, 16), (1, 32, 8, 1, 128, 0, 131072, 12, 24), (1, 32, 8, 1, 128, 1, 32768, 12, 16),
    (1, 32, 8, 1, 128, 1, 131072, 16, 32), (1, 8, 8, 1, 32, 1, 32768, 6, 16), (1, 16, 16, 1, 64, 0, 16385, 4, 12),
    (2, 32, 8, 1, 128, 0, 8192, 6, 8), (1, 32, 8, 4, 128, 1, 32771, 12, 16), (1, 8, 1, 1, 128, 0, 32768, 12, 32)])
def test_rule_for_few_rows_of_long_sequences(plan, batch, heads, kv, tokens, d, bits8, keys, least, most):
    # The waves divide the keys, and the splits are among those measured within a
    # fifth of the best; tiled kernels took 5 to 65% longer, most other splits more.
    kernel, splits, *_ = plan(batch, heads, kv, tokens, d, bits8, keys)
    assert kernel == KEYS and least <= splits <= most
