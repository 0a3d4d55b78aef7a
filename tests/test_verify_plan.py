"""The rules by which draft verification is launched, as a host program runs them
(csrc/launch_plan.h), and the calls that one launch does not take."""
import ctypes
import random

import pytest

from frisk_amd import runtime as rt
from tests.test_more_ops_capi import call, verify_desc
from tests.test_tree_plan import program

CUS = 256


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """(pieces, segments, alone, workgroups with tables, limits ...) of calls (batch, tokens, vocab, bytes)."""
    run = program(tmp_path_factory, "verify", f"""
using namespace frisk::plan;
int main(int, char** v) {{
  FILE* f = fopen(v[1], "r");
  long long b, t, n;
  int bytes;
  while (fscanf(f, "%lld %lld %lld %d", &b, &t, &n, &bytes) == 4) {{
    const VerifyPlan p = verify_plan(b, t, n, bytes);
    printf("%d %lld %d %lld %lld %lld %lld %d %lld %lld\\n", p.pieces, (long long)p.segments,
           (int)verify_alone(b, t, p.segments, {CUS}), (long long)verify_tables(b, t, p.segments, {CUS}),
           (long long)kVerifyShort, (long long)kVerifyAlone, (long long)kVerifyTrees, kVerifyTableWaves,
           (long long)kVerifySegments, (long long)kVerifyNodes * 52);
  }}
  fclose(f);
}}""")
    path = tmp_path_factory.mktemp("calls") / "calls"

    def of(calls):
        path.write_text("\n".join(" ".join(map(str, c)) for c in calls))
        return run(path)
    return of


def test_segments_cover_every_row(plan):
    # A row begins up to N - 1 elements before its first piece of 16 bytes; its tail is shorter
    # than a piece and has 32 lanes, its head the other 32.
    vocabs = [*range(1, 1100), *(k * 1024 + d for k in (1, 2, 4, 8, 16, 33, 64, 65) for d in range(-9, 10)),
              32000, 50257, 131072, (1 << 24) - 1, 1 << 24]
    calls = [(b, t, v, e) for v in vocabs if v > 0 for e in (2, 4) for b, t in ((1, 1), (300, 1), (8, 6), (64, 64))]
    for (b, t, v, e), (pieces, segments, *_) in zip(calls, plan(calls)):
        n = 16 // e
        assert pieces in (1, 4) and segments >= 1
        for head in range(n):
            full = (v - min(head, v)) // n
            assert segments * 64 * pieces >= full
        # No segment but the first is empty.
        assert segments == 1 or (segments - 1) * 64 * pieces < v // n


def test_launches_fit_their_memory_and_grids(plan):
    rng = random.Random(3)
    calls = [(b, t, v, e) for b in (1, 2, 31, 32, 64, 128, 200, 256, 1000) for t in (1, 2, 8, 64, 1024)
             for v in (1, 500, 8000, 8192, 8193, 32000, 49152, 131072) for e in (2, 4)]
    calls += [(int(2 ** rng.uniform(0, 22)), int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(0, 24)), rng.choice([2, 4]))
              for _ in range(4000)]
    taken = {"alone": 0, "short": 0, "tables": 0, "three": 0}
    for (b, t, v, e), row in zip(calls, plan(calls)):
        pieces, segments, alone, tables, short, most, trees, table_waves, limit, walk_lds = row
        assert walk_lds <= 64 * 1024 - 4096
        if b > trees or b * t * segments > limit:
            continue
        groups = -(-segments // 4)
        if alone:
            # Its rests are in LDS, and one launch has a workgroup of 1024 a tree.
            assert t == 1 and segments <= most and b * 1024 < 2 ** 32
            taken["alone"] += 1
            continue
        assert b * t * groups * 256 < 2 ** 32 and b * 1024 < 2 ** 32
        if t > 1:
            if tables:
                assert 1 <= tables <= -(-segments // table_waves)
                assert b * t * tables * table_waves * 64 < 2 ** 32
                taken["tables"] += 1
            if pieces == 1 and segments <= short:
                taken["short"] += 1
            else:
                taken["three"] += 1
                # (One piece a lane is for rows that a wave's lanes take at once.)
                assert pieces == 4 or segments <= 64
    assert all(n > 20 for n in taken.values()), taken


@pytest.mark.parametrize("tokens,vocab,dtype", [(1, 100, rt.BF16), (3, 100, rt.F32), (1, 8000, rt.F16)])
def test_more_trees_than_a_launch_takes(tokens, vocab, dtype):
    # A tree has a workgroup of 1024 threads, in the walk or by itself: 2^22 trees have 2^32.
    lib = rt.load()
    sizes = dict(tokens=tokens, vocab=vocab, dtype=dtype, logits=1 << 40)
    for batch in (1 << 22, (1 << 22) + 1, ((1 << 24) - 1) // (tokens * 16)):
        d = verify_desc(batch=batch, workspace_bytes=1 << 40, workspace=1 << 46, **sizes)
        fits = batch < 1 << 22
        assert (lib.frisk_tree_verify_workspace_size(ctypes.byref(d)) >= 0) == fits, batch
        if not fits:
            rc, err = call("frisk_tree_verify", d)
            assert rc == rt.EUNSUP and err.startswith("frisk_tree_verify: more "), err
