"""More of the packed prompt attention and the page operators: pages that a row has lost,
tables of the greatest width, rows before the first sequence, bounds of many sequences
that fall or lead out, keys that are not finite.

Checks of the kernels' sources on the CPU run in processes of their own, as in
test_packed_lanes."""

from __future__ import annotations

import ctypes
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))

from test_packed_lanes import (  # noqa: E402, F401
    CSRC, LANES, MORE, POOLS, REPO, Kernels, _compiler, _packed, formula, lanes_library, state_of)
from test_packed import Pool, Prompts, built, gpu, ints, near  # noqa: E402

from qwen_int4_hip import (  # noqa: E402
    _lib, packed_attention_hip, paged_append_hip, paged_attention_hip, paged_compact_hip, paged_fork_hip, paged_resize_hip)

BF16, F16, I32 = torch.bfloat16, torch.float16, torch.int32
WILD = [2 ** 31 - 1, -(2 ** 31)]


def _lists(*tensors):
    return tuple(t.tolist() for t in tensors)


def resized_cached(table, lengths, users, page, cached):
    """The resize's answers, entry by entry: one that holds cached positions is given no page."""
    table, users, missing = [list(r) for r in table], list(users), []
    free = iter([p for p, n in enumerate(users) if n == 0])
    for row, length, filled in zip(table, lengths, cached):
        need = -(-max(length, 0) // page)
        for c, e in enumerate(row):
            named = 0 <= e < len(users)
            if c >= need:
                if named:
                    users[e] -= 1
                row[c] = -1
            elif not named:
                row[c] = -1 if c * page < filled else next(free, -1)
                if row[c] >= 0:
                    users[row[c]] += 1
        missing.append(need - sum(e >= 0 for e in row))
    return table, users, missing


def _lengths(seed, batch, most):
    return torch.randint(0, most + 1, (batch,), generator=torch.Generator().manual_seed(seed)).tolist()


def cached_cases(sizes, wild, spare):
    """(table, users, [(lengths, cached), ...]) of rows some of whose entries name no page."""
    batch, width, pages, page = sizes
    table, lengths, users = state_of(11, *sizes, spare=spare, wild=wild)
    for b in range(0, batch, 2):  # an entry is lost here and there
        c = (7 * b) % width
        if 0 <= table[b][c] < pages:
            users[table[b][c]] -= 1
            table[b][c] = -1
    most = width * page + 20
    return table, users, [(_lengths(1, batch, most), lengths), (_lengths(2, batch, most), _lengths(3, batch, most)),
                          ([width * page] * batch, [page * (width // 2) + b % 3 for b in range(batch)]),
                          (lengths, [(0, -5, *WILD)[b % 4] for b in range(batch)])]


# ---------------------------------------------------------------------------
# On the CPU, in the process of a check
# ---------------------------------------------------------------------------

class MoreKernels(Kernels):
    def resize_cached(self, table, lengths, users, page, cached):
        (batch, width), pages = table.shape, len(users)
        answers = self.empty(batch, width), self.empty(pages), self.empty(batch)
        need = self.lib.qwen2_paged_resize_workspace_bytes(batch, width, pages)
        workspace = self.memory(torch.full((need,), 0xA5, dtype=torch.uint8))
        self.check(self.lib.qwen2_paged_resize_cached(
            table.data_ptr(), width, lengths.data_ptr(), cached.data_ptr(), users.data_ptr(),
            *(t.data_ptr() for t in answers), batch, width, pages, page, workspace.data_ptr(), need, None))
        return answers


def _lost(kernels):
    """A fork finds no free page for its second child while a sequence ends and gives one up:
    the next resize does not pass that one off as the child's."""
    k, v = (kernels.memory(torch.zeros(1, 3, 1, 16, 8, dtype=BF16)) for _ in range(2))
    table, lengths, users, missing = kernels.fork(k, v, kernels.ints([[0, 1, -1], [2, -1, -1]]), kernels.ints([20, 16]),
                                                  kernels.ints([1, 1, 1]), kernels.ints([0, 0]))
    assert _lists(table, lengths, users, missing) == ([[0, 1, -1], [0, -1, -1]], [20, 20], [2, 1, 0], [0, 1])
    for _ in range(2):  # at every call, as the row grows
        table, users, missing = kernels.resize_cached(table, kernels.ints([20, 21]), users, 16, lengths)
        assert _lists(table, users, missing) == ([[0, 1, -1], [0, -1, -1]], [2, 1, 0], [0, 1])
        lengths = kernels.ints([20, 21])
    # a new page behind the lost one is given; freed, the row starts anew
    grown = kernels.resize_cached(table, kernels.ints([20, 40]), users, 16, lengths)
    assert _lists(*grown) == ([[0, 1, -1], [0, -1, 2]], [2, 1, 1], [0, 1])
    table, users, missing = kernels.resize_cached(table, kernels.ints([20, 0]), users, 16, lengths)
    assert _lists(table, users, missing) == ([[0, 1, -1], [-1, -1, -1]], [1, 1, 0], [0, 0])
    anew = kernels.resize_cached(table, kernels.ints([20, 5]), users, 16, kernels.ints([20, 0]))
    assert _lists(*anew) == ([[0, 1, -1], [2, -1, -1]], [1, 1, 1], [0, 0])


def _cached(kernels):
    for sizes in [s for s in POOLS if s[2] < 400] + [(3, 20, 16500, 16), (2, 4200, 500, 16)]:
        for wild in (False, True):
            table, users, calls = cached_cases(sizes, wild, min(sizes[2] // 7, 9))
            for lengths, cached in calls:
                got = kernels.resize_cached(kernels.ints(table), kernels.ints(lengths), kernels.ints(users), sizes[3],
                                            kernels.ints(cached))
                assert _lists(*got) == resized_cached(table, lengths, users, sizes[3], cached), (sizes, wild)


def _ends(kernels):
    """The last 640 columns of rows as wide as can be: kept, given up, and (by a page size that makes
    a length need them) given."""
    call = kernels.lib.ends_resize
    call.restype, call.argtypes = None, [ctypes.c_void_p] * 5 + [ctypes.c_int64] * 2 + [ctypes.c_int] * 4
    pages, count = 700, 640
    for width in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 63, 2 ** 31 - 64, 2 ** 31 - 300, 2 ** 30, 1000):
        start = width - count
        for length, shift in ((2 ** 31 - 1, 0), (start + 5, 0), (0, 4)):
            row = [(7 * c) % pages if c % 3 else -1 for c in range(count)]
            table, new_table, said = kernels.ints(row), kernels.empty(count), kernels.empty(2)
            users, spare = kernels.ints([1] * pages), [pages - 1 - c for c in range(100)]
            call(table.data_ptr(), new_table.data_ptr(), users.data_ptr(), kernels.ints(spare).data_ptr(), said.data_ptr(),
                 width, start, pages, 100, length, shift)
            upto, want, after, given = min(length, width) - start if length else 0, [], [1] * pages, iter(spare)
            for c, e in enumerate(row):
                if c >= upto:
                    if e >= 0:
                        after[e] -= 1
                    e = -1
                elif e < 0:
                    e = next(given, -1)
                    if e >= 0:
                        after[e] += 1
                want.append(e)
            assert new_table.tolist() == want and users.tolist() == after, (width, length)
            assert said.tolist() == [sum(e < 0 for e in row[:max(upto, 0)]), sum(e >= 0 for e in want)]


def _before(kernels):
    """Sequences that begin behind the first row: the rows before them are as those behind the last."""
    for first, lengths, tail in ((1, [2, 0, 3], 0), (3, [40, 7], 2), (70, [33], 1), (5, [1 + b % 2 for b in range(100)], 3)):
        rows = first + sum(lengths)
        q, k, v, _ = _packed(kernels, [rows], 4, 2, 64, tail=tail)
        cu = kernels.ints([first + sum(lengths[:b]) for b in range(len(lengths) + 1)])
        want = formula(q, k, v, cu)
        for zero_rest, rest in ((1, 0.0), (0, 7.0)):
            out = kernels.attention(q, k, v, cu, zero_rest, fill=7.0)
            assert bool((out[:first] == rest).all()) and bool((out[rows:] == rest).all()), (first, zero_rest)
            # (a half step of the output and of each probability, values of a few units)
            assert float((out.double() - want)[first:rows].abs().amax()) < 4 * torch.finfo(BF16).eps
    for values in [[5, 2], [9, 9], [2 ** 31 - 1, 3], [4, -1], [-3, 2]]:  # rows of 8
        q, k, v, _ = _packed(kernels, [8], 4, 2, 64)
        out = kernels.attention(q, k, v, kernels.ints(values), fill=7.0)
        end = min(max(values[1], 0), 8)
        assert not out[:min(max(values[0], 0), end)].any() and not out[end:].any(), values


def wild_bounds(batch, rows):
    """Row bounds of `batch` sequences that no program should have."""
    even = [rows * b // batch for b in range(batch + 1)]
    gen = torch.Generator().manual_seed(batch)
    anywhere = torch.randint(-3, rows + 4, (batch + 1,), generator=gen).tolist()
    return [even[::-1], [rows] * (batch + 1), [0, rows] * (batch // 2) + [0] * (batch % 2 + 1), [WILD[0]] * (batch + 1),
            [WILD[1]] * (batch + 1), [WILD[b % 2] for b in range(batch + 1)], anywhere, [*anywhere[:-1], rows],
            [*anywhere[:-1], -1], [*even[:batch // 2], WILD[0], *even[batch // 2 + 1:]], [0] * batch + [rows],
            [0] * (batch - 1) + [rows, 2]]


def _many_bounds(kernels):
    for batch in (65, 256, 257, 300):
        rows = 70
        q, k, v, _ = _packed(kernels, [rows], 2, 1, 64)
        for values in wild_bounds(batch, rows):
            end = min(max(values[-1], 0), rows)
            out = kernels.attention(q, k, v, kernels.ints(values), 0, fill=7.0)
            assert bool((out[end:] == 7.0).all()), (batch, values[:5])
            out = kernels.attention(q, k, v, kernels.ints(values), 1, fill=7.0)
            assert not out[end:].any(), (batch, values[:5])


def pieces(bounds, rows, group, kv_heads, tile_rows):
    """(first row, (token, head) rows, tile, head) of every workgroup, sequences in order, last tiles first."""
    end = min(max(bounds[-1], 0), rows)
    found = []
    for first, last in zip(bounds, bounds[1:]):
        first = min(max(first, 0), end)
        count = (min(max(last, first), end) - first) * group
        found += [(first, count, tile, head) for tile in reversed(range(-(-count // tile_rows))) for head in range(kv_heads)]
    return found


def _finds(kernels):
    """Every workgroup's place, and that those past the last one have none."""
    call = kernels.lib.finds
    call.restype, call.argtypes = None, [ctypes.c_void_p] * 2 + [ctypes.c_int] * 7
    for batch, rows, group, kv_heads, tile_rows in ((1, 300, 6, 2, 64), (2, 90, 1, 1, 32), (63, 400, 7, 1, 32), (64, 5000, 6, 2, 128),
                                                    (65, 500, 3, 2, 64), (256, 900, 1, 1, 32), (257, 2000, 2, 1, 64),
                                                    (300, 600, 6, 2, 128), (1100, 3000, 1, 3, 64)):
        for values in [[rows * b // batch for b in range(batch + 1)]] + (wild_bounds(batch, rows) if batch > 1 else []):
            want = pieces(values, rows, group, kv_heads, tile_rows)
            if len(want) > 3000:
                continue
            some = len(want) + 3
            for longest in ((1, 2) if batch <= 64 else (0,)):
                said = kernels.empty(some, 5)
                call(kernels.ints(values).data_ptr(), said.data_ptr(), batch, rows, group, kv_heads, tile_rows, longest, some)
                got = said.tolist()
                assert [g[0] for g in got] == [1] * len(want) + [0] * 3, (batch, values[:5])
                got = [tuple(g[1:]) for g in got[:len(want)]]
                assert got == want if longest == 0 else sorted(got) == sorted(want), (batch, longest, values[:5])
                if longest == 1:  # (the most keys first)
                    assert [g[2] for g in got] == sorted((g[2] for g in got), reverse=True)


CHECKS = {"lost": _lost, "cached": _cached, "ends": _ends, "before": _before, "many_bounds": _many_bounds, "finds": _finds}


@pytest.fixture(scope="module")
def more_library(lanes_library):  # noqa: F811
    """The library of test_packed_lanes, with the drivers of lanes_more in it."""
    root = lanes_library.parent
    library = root / "more.so"
    drivers = [(source, root / f"more_{source.stem}.o") for source in sorted(MORE.glob("*.cpp"))]
    for source, made in drivers:
        subprocess.run([_compiler(), "-std=c++17", "-O2", "-fPIC", "-ffp-contract=off", "-mf16c", "-mfma", "-w", f"-I{LANES}",
                        f"-I{root}", f"-I{REPO / 'include'}", f"-I{MORE}", "-include", str(MORE / "more.h"), "-x", "c++", "-c",
                        str(source), "-o", str(made)], check=True)
    # (a driver brings its kernels' source with it: their entry points come once)
    rest = [made for made in root.glob("*.o") if made.name not in ("qwen2_pages.o", "qwen2_packed_attention.o")]
    subprocess.run([_compiler(), "-shared", *map(str, rest), "-o", str(library)], check=True)
    return library


@pytest.mark.parametrize("side", ["end", "start"])
@pytest.mark.parametrize("name", CHECKS)
def test_on_the_cpu(more_library, name, side):
    result = subprocess.run([sys.executable, __file__, str(more_library), name, side], capture_output=True, text=True,
                            timeout=600)
    assert result.returncode == 0 and result.stdout.endswith("done\n"), (result.returncode, result.stderr[-2000:])


PARTS_PROGRAM = r"""
#define __host__
#define __device__
#include "qwen2_pages.h"
#include <cstdio>
using namespace w4g64;
int main() {
    const int64_t spans[][2] = {{1, 1100}, {1 << 30, (1 << 30) + 1}, {2147483648ll - 1100, 2147483648ll}};
    for (const auto& span : spans)
        for (int64_t w = span[0]; w < span[1]; ++w)
            for (int p = 0; p < 8; ++p) {
                const ColumnPart part = column_part((int)w, p, 8);
                printf("%d %d %d\n", (int)w, part.from, part.end);
            }
}
"""


def test_the_parts_of_a_row_cover_it(tmp_path):
    """At every width one after the other, without a gap, from multiples of 64 on."""
    source, program = tmp_path / "parts.cpp", tmp_path / "parts"
    source.write_text(PARTS_PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(source), "-o", str(program)], check=True)
    said = [tuple(map(int, line.split())) for line in subprocess.run([str(program)], check=True, capture_output=True,
                                                                     text=True).stdout.splitlines()]
    assert len(said) == 8 * (1099 + 1 + 1100)
    for at in range(0, len(said), 8):
        width, reached = said[at][0], 0
        for w, begin, end in said[at:at + 8]:
            assert w == width and begin == reached and end >= begin and (begin % 64 == 0 or begin == width)
            reached = end
        assert reached == width


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------

@built
def test_cached_is_refused_before_launch():
    table, lengths, users = torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32), torch.zeros(6, dtype=I32)
    for cached, error, said in [(lengths.long(), TypeError, "cached must have dtype torch.int32"),
                                (torch.zeros(3, dtype=I32), ValueError, r"cached must have shape \[2\]"),
                                (table, ValueError, "cached must have 1 dimensions"), ([0, 0], TypeError, "must be a torch.Tensor"),
                                (lengths, ValueError, "must be a GPU tensor")]:
        with pytest.raises(error, match=said):
            paged_resize_hip(table, lengths, users, page_size=16, cached=cached)
    buffer = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buffer) + 15) & ~15
    call = _lib.load().qwen2_paged_resize_cached
    assert call(p, 3, p, p + 2, p, p, p, p, 2, 3, 6, 16, None, 0, None) == 1
    assert call(p, 3, p, p, p, p, p, p, 2, 3, 6, 24, None, 0, None) == 1


# ---------------------------------------------------------------------------
# On the GPU
# ---------------------------------------------------------------------------

@gpu
def test_refusals_come_before_any_copy():
    """Arguments that a good call would copy (unaligned rows, strided indices) are not when it is refused."""
    def odd(*shape):
        return torch.zeros(2 * math.prod(shape) + 3, dtype=BF16, device="cuda")[3:3 + math.prod(shape)].view(shape)

    cu, one = torch.zeros(3, 2, dtype=I32, device="cuda")[:, 0], torch.zeros(5, 2, 64, dtype=BF16, device="cuda")
    far = torch.zeros(2, 1 << 25, dtype=BF16, device="cuda")[:, :128].view(2, 2, 64)
    table, lengths = torch.zeros(2, 6, dtype=I32, device="cuda")[:, ::2], torch.zeros(2, 2, dtype=I32, device="cuda")[:, 0]
    users, pool = torch.zeros(6, 2, dtype=I32, device="cuda")[:, 0], torch.zeros(2, 6, 2, 24, 64, dtype=BF16, device="cuda")
    heads = [odd(5, 4, 48), odd(5, 2, 48), odd(5, 2, 48)]
    calls = [
        (ValueError, "head_dim of 64 or 128", packed_attention_hip, (*heads, cu), {}),
        (ValueError, "head_dim of 64 or 128", packed_attention_hip, (*heads, cu[:1]), {}),
        (ValueError, "multiple of kv_heads", packed_attention_hip, (odd(5, 3, 64), one, one, cu), {}),
        (ValueError, "multiple of kv_heads", packed_attention_hip, (odd(5, 3, 64)[:0], one[:0], one[:0], cu), {}),
        (ValueError, "finite", packed_attention_hip, (odd(5, 4, 64), one, one, cu), {"scale": math.nan}),
        (ValueError, "2\\^24 elements apart", packed_attention_hip, (odd(2, 4, 64), far, far, cu), {}),
        (ValueError, "power of two", paged_resize_hip, (table, lengths, users), {"page_size": 24}),
        (ValueError, "power of two", paged_resize_hip, (table, lengths, users), {"page_size": 24, "cached": lengths}),
        (ValueError, "power of two", paged_fork_hip, (pool[0], pool[1], table, lengths, users, lengths), {}),
        (ValueError, "power of two", paged_compact_hip, (pool[0], pool[1], table, users), {}),
    ]
    for error, said, call, args, more in calls:
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        with pytest.raises(error, match=said):
            call(*args, **more)
        assert torch.cuda.memory_stats()["allocation.all.allocated"] == before, (call, said)


@gpu
@pytest.mark.parametrize("wild", [False, True])
@pytest.mark.parametrize("sizes", POOLS + [(300, 40, 5000, 16), (9, 5000, 70000, 32), (1100, 7, 3000, 16)])
def test_resize_gives_no_page_to_cached_positions(sizes, wild):
    page = sizes[3]
    table, users, calls = cached_cases(sizes, wild, min(sizes[2] // 7, 9))
    device = ints(table).view(sizes[0], -1), ints(users)
    for lengths, cached in calls:
        got = paged_resize_hip(device[0], ints(lengths), device[1], page_size=page, cached=ints(cached))
        assert _lists(*got) == resized_cached(table, lengths, users, page, cached)
        strided = torch.stack((ints(cached), ints(cached)), 1)[:, 1]
        assert _lists(*paged_resize_hip(device[0], ints(lengths), device[1], page_size=page, cached=strided)) == _lists(*got)
        none = paged_resize_hip(device[0], ints(lengths), device[1], page_size=page, cached=ints([0] * sizes[0]))
        assert _lists(*none) == _lists(*paged_resize_hip(device[0], ints(lengths), device[1], page_size=page))


@gpu
def test_a_lost_page_stays_missing_in_a_graph():
    p = Pool(12, 12, 9, 150, 16, layers=1)
    table, _, users = p.indices()
    table[3, 0] = -1
    lengths, cached = ints(p.lengths), ints(p.lengths)
    paged_resize_hip(table, lengths, users, page_size=16, cached=cached)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_resize_hip(table, lengths, users, page_size=16, cached=cached)
    for turn in range(4):
        lengths.copy_(ints(_lengths(turn, 12, 9 * 16)))
        cached.copy_(ints(_lengths(turn + 9, 12, 9 * 16)))
        graph.replay()
        torch.cuda.synchronize()
        assert _lists(*got) == resized_cached(table.tolist(), lengths.tolist(), users.tolist(), 16, cached.tolist())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_row_that_lost_a_page_is_not_served_from_another_one(dtype):
    """Two sequences, one forked into three children while the other ends and no page is free: the
    pages that the ended one gave up go to no lost place, so that the children without a copy
    attend NaN at every step, and the one that kept its page what the formula says."""
    heads, kv_heads, dim, page = 4, 2, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(5)
    k_pages, v_pages = (torch.randn(5, kv_heads, page, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    users, table, lengths = ints([1, 1, 1, 1, 1]), ints([[4, 1, 2, -1], [3, 0, -1, -1]]), ints([37, 30])
    keys, values = (torch.cat([t[p].transpose(0, 1) for p in (4, 1, 2)])[:37].clone() for t in (k_pages, v_pages))
    table, lengths, users, lost = paged_fork_hip(k_pages, v_pages, table, lengths, users, ints([0, 0, 0]))
    assert lost.tolist() == [0, 1, 1] and users.tolist() == [0, 3, 1, 0, 3]
    cu = ints([0, 1, 2, 3])
    for step in range(11):  # to the end of the last page
        table, users, missing = paged_resize_hip(table, lengths + 1, users, page_size=page, cached=lengths)
        lengths = lengths + 1
        assert missing.tolist() == [0, 1, 1] and table[1:, 2].tolist() == [-1, -1]
        q, k, v = (torch.randn(3, n, dim, generator=gen, device="cuda").to(dtype) for n in (heads, kv_heads, kv_heads))
        rotated = paged_append_hip(q, k, v, k_pages, v_pages, table, cu, lengths, None)
        got = paged_attention_hip(rotated, k_pages, v_pages, table, cu, lengths).double()
        assert bool(got[1:].isnan().all())
        keys, values = torch.cat((keys, k[:1])), torch.cat((values, v[:1]))
        for h in range(heads):
            w = torch.softmax(keys[:, h // 2].double() @ q[0, h].double() * dim ** -0.5, 0)
            want = w @ values[:, h // 2].double()
            # (a half step of the result, values of a few units, and one of each probability's two terms)
            assert float((got[0, h] - want).abs().amax()) < 4 * torch.finfo(dtype).eps
    lengths[1:] = 0
    table, users, missing = paged_resize_hip(table, lengths, users, page_size=page, cached=lengths)
    assert not missing.any() and sorted(users.tolist()) == [0, 0, 1, 1, 1] and bool((table[1:] == -1).all())


@gpu
def test_page_operators_over_a_row_as_wide_as_can_be():
    """2^31 - 1 columns, more than any length needs; pages named in the last of them are given up
    (resize, fork) or renamed (compact)."""
    width, pages = 2 ** 31 - 1, 100
    table = torch.full((1, width), -1, dtype=I32, device="cuda")
    last = [0, 1, 5, width // 2, width - 700, width - 513, width - 512, width - 257, width - 64, width - 2, width - 1]
    table[0, last] = ints(range(20, 20 + len(last)))
    users = torch.zeros(pages, dtype=I32, device="cuda")
    users[20:20 + len(last)] = 1
    got = paged_resize_hip(table, ints([40]), users, page_size=16)
    assert got[0].shape == (1, width) and got[0][0, :4].tolist() == [20, 21, 0, -1] and int((got[0] >= 0).sum()) == 3
    assert int((got[0] == -1).sum()) == width - 3 and got[2].tolist() == [0]
    assert got[1].tolist() == [int(p in (0, 20, 21)) for p in range(pages)]
    del got
    pools = [torch.zeros(pages, 1, 16, 8, dtype=BF16, device="cuda") for _ in range(2)]
    got = paged_fork_hip(*pools, table, ints([32]), users, ints([0]))
    assert got[0][0, :3].tolist() == [20, 21, -1] and int((got[0] == -1).sum()) == width - 2
    assert got[1].tolist() == [32] and got[3].tolist() == [0] and got[2].tolist() == [int(p in (20, 21)) for p in range(pages)]
    del got
    got = paged_compact_hip(*pools, table, users)
    assert got[0][0, last].tolist() == list(range(len(last))) and int((got[0] == -1).sum()) == width - len(last)
    assert got[1].tolist() == [int(p < len(last)) for p in range(pages)]


@gpu
@pytest.mark.parametrize("batch", [65, 256, 257, 300])
def test_bounds_of_many_sequences_stay_in_the_buffers(batch):
    rows = 700
    p = Prompts([rows], heads=6)
    for values in wild_bounds(batch, rows):
        p.cu = ints(values)
        out = torch.full_like(p.q, 7.0)
        p.attention(out=out)
        end = min(max(values[-1], 0), rows)
        assert bool((out[end:] == 7.0).all()) and not p.attention()[end:].any()


@gpu
@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("lengths, heads", [([20, 30], 4), ([5, 400, 70], 4), ([300], 40), ([130] * 30, 12), ([290] * 30, 12),
                                            ([25] * 80, 4)])
def test_keys_that_are_not_finite(dtype, dim, bad, lengths, heads):
    """Infinite elements of two keys: a score of +inf leaves its row NaN, one of -inf leaves its key
    out (and a row that sees no other one NaN); whole keys besides, whose scores have no sum."""
    at, half = lengths[0] if len(lengths) > 1 else 0, torch.finfo(dtype).eps / 2
    for whole in (False, True):
        p = Prompts(lengths, heads=heads, kv_heads=2, dim=dim, dtype=dtype)
        for spot in (at, at + 11):
            p.k[spot, :, slice(None) if whole else 5] = bad
        want, begin = torch.zeros(p.q.shape, dtype=torch.float64, device="cuda"), 0
        slack = want.clone()
        for n in lengths:
            x, y, z = (t[begin:begin + n].double().transpose(0, 1).repeat_interleave(heads // t.shape[1], 0) for t in (p.q, p.k, p.v))
            hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
            w = torch.softmax((x @ y.transpose(1, 2) * dim ** -0.5).masked_fill(hidden, -math.inf), dim=-1)
            part, size = w @ z, w @ z.abs()
            # as Prompts.reference() bounds it, by the scores that are finite
            big = (x.abs() @ y.abs().nan_to_num(posinf=0).transpose(1, 2)).amax() * dim ** -0.5
            off = 2.0 ** -24 * (2 * (dim + 8) * big + n / 4 + 64) * size + half * (1 + 2 * half) * (size + part.abs())
            want[begin:begin + n] = part.transpose(0, 1)
            slack[begin:begin + n] = (off + n * 2.0 ** -36 * z.abs().amax()).transpose(0, 1)
            begin += n
        near(p.attention(), want, slack)


@gpu
@pytest.mark.parametrize("first, lengths, more", [
    (1, [2, 0, 1], {}), (70, [200, 9], {"heads": 6}), (3, [600], {"heads": 12, "dim": 128}),
    (400, [1300, 40], {"heads": 12, "dim": 128, "dtype": F16}), (37, [1 + b % 9 for b in range(90)], {})])
def test_rows_before_the_first_sequence(first, lengths, more):
    p = Prompts([first, *lengths], tail=2, **more)
    want, slack = p.reference()
    want[:first] = 0
    bounds = p.cu[1:].clone()
    torch.full_like(p.q, 7.0)  # (what an answer's memory held)
    got = packed_attention_hip(p.q, p.k, p.v, bounds)
    near(got, want, slack)
    assert not got[:first].any() and not got[p.total:].any()
    out = torch.full_like(got, 7.0)
    packed_attention_hip(p.q, p.k, p.v, bounds, out=out)
    assert torch.equal(out[first:p.total], got[first:p.total])
    assert bool((out[:first] == 7.0).all()) and bool((out[p.total:] == 7.0).all())


if __name__ == "__main__":
    torch.set_num_threads(1)
    CHECKS[sys.argv[2]](MoreKernels(sys.argv[1], sys.argv[3]))
    print("done")
