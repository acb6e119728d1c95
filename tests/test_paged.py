"""The paged serving operators (qwen_int4_hip.paged) against plain
implementations in 64 bits, and what they refuse.

Tolerances count roundings: a result in 16 bits is off by at most
finfo.eps / 2 of its value, and what fp32 adds before it is bounded beside each
comparison from the sums that the reference forms."""

from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

import qwen_int4_hip
from qwen_int4_hip import _lib, paged_append_hip, paged_attention_hip, verify_drafts_hip

REPO = Path(__file__).resolve().parents[1]
CSRC = REPO / "qwen2-int4-systems_amd" / "csrc"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

built = pytest.mark.skipif(not _lib.library_built(), reason="HIP library not built (run __graft_entry__.build())")


def gpu(test):
    return pytest.mark.gpu(pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a ROCm GPU")(built(test)))


# ---------------------------------------------------------------------------
# On the CPU: the index arithmetic of the kernels, and the refusals
# ---------------------------------------------------------------------------

INDEX_PROGRAM = r"""
#define __host__
#define __device__
#include "qwen2_paged.h"
#include <cstdio>
using namespace w4g64;
int main() {
    const int32_t table[4] = {3, -1, 7, 0};
    // pages 0 .. 6 exist: entry 2 names none; entry 1 is unset
    const int64_t positions[] = {0, 15, 16, 32, 47, 48, 63, 64, -1, 1LL << 40, -(1LL << 40)};
    for (int64_t p : positions) printf("%d ", page_of(table, 4, 4, 7, p));
    const int32_t lengths[3] = {10, 2, -5};
    const int32_t fine[4] = {0, 3, 3, 8}, wild[4] = {-7, 90, 2, -1};
    for (int b = 0; b < 3; ++b) {
        const SequenceRows s = sequence_rows(fine, lengths, b, 8), w = sequence_rows(wild, lengths, b, 8);
        printf("| %d %d %lld / %d %d %lld ", s.begin, s.end, (long long)s.first, w.begin, w.end, (long long)w.first);
    }
}
"""


def test_indices_from_device_memory_stay_in_bounds(tmp_path):
    source, program = tmp_path / "index.cpp", tmp_path / "index"
    source.write_text(INDEX_PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(source), "-o", str(program)], check=True)
    said = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout
    pages, *rows = said.split("|")
    assert pages.split() == ["3", "3", "-1", "-1", "-1", "0", "0", "-1", "-1", "-1", "-1"]
    assert [r.split() for r in rows] == [
        ["0", "3", "7", "/", "0", "8", "2"],    # three rows after seven; -7 .. 90 is every row
        ["3", "3", "2", "/", "8", "8", "2"],    # none; 90 .. 2 none
        ["3", "8", "-10", "/", "2", "2", "-5"]]  # a length below its rows: negative positions


REST_PROGRAM = r"""
#define __host__
#define __device__
#include "qwen2_paged.h"
#include <cstdio>
using namespace w4g64;
int main() {
    const int32_t ends[] = {0, 3, 8, 9, 2147483647, -1, -2147483647 - 1};
    for (int32_t end : ends) {
        const int32_t cu[3] = {0, 0, end};
        printf("%d", rows_end(cu, 2, 8));
        const unsigned workgroups[] = {0, 1, 5, 2147483646};
        for (unsigned workgroup : workgroups) {  // rows behind the last sequence, of all 8
            const int64_t r = rest_row(cu, 2, 8, workgroup);
            if (r < 8) printf(" %lld", (long long)r);
        }
        printf("|");
    }
}
"""


def test_rows_behind_the_last_sequence_stay_in_bounds(tmp_path):
    source, program = tmp_path / "rest.cpp", tmp_path / "rest"
    source.write_text(REST_PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(source), "-o", str(program)], check=True)
    said = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout
    assert [part.split() for part in said.split("|")[:-1]] == [
        ["0", "0", "1", "5"], ["3", "3", "4"], ["8"], ["8"], ["8"], ["0", "0", "1", "5"], ["0", "0", "1", "5"]]


def _arguments(device="cpu", dtype=BF16, rows=5, heads=4, kv_heads=2, dim=64, page=16, pages=6, batch=2, width=3):
    def t(*shape, dtype=dtype):
        return torch.zeros(shape, dtype=dtype, device=device)

    cache = {"k_pages": t(pages, kv_heads, page, dim), "v_pages": t(pages, kv_heads, page, dim),
             "page_table": t(batch, width, dtype=torch.int32), "cu_rows": t(batch + 1, dtype=torch.int32),
             "lengths": t(batch, dtype=torch.int32)}
    append = {"q": t(rows, heads, dim), "k": t(rows, kv_heads, dim), "v": t(rows, kv_heads, dim), **cache,
              "inv_freq": t(dim // 2, dtype=F32)}
    return append, {"q": t(rows, heads, dim), **cache}


BAD_CACHE = [
    ({"k_pages": torch.zeros(6, 2, 16, 64)}, TypeError, "k_pages must have dtype"),
    ({"v_pages": torch.zeros(6, 2, 16, 64, dtype=F16)}, TypeError, "v_pages must have the dtype"),
    ({"v_pages": torch.zeros(6, 2, 32, 64, dtype=BF16)}, ValueError, "v_pages must have the shape"),
    ({"k_pages": torch.zeros(6, 2, 16 * 64, dtype=BF16)}, ValueError, "k_pages must have 4 dimensions"),
    ({"k_pages": torch.zeros(6, 2, 64, 16, dtype=BF16).transpose(2, 3)}, ValueError, "k_pages must be 16-byte"),
    ({"v_pages": torch.zeros(6, 2, 16, 68, dtype=BF16)[..., :64]}, ValueError, "v_pages must be 16-byte"),
    ({"k_pages": torch.zeros(2 * 2 * 16 * 64 * 6 + 8, dtype=BF16)[4:6 * 2048 + 4].view(6, 2, 16, 64)}, ValueError,
     "k_pages must be 16-byte"),
    ({"k_pages": torch.zeros(1, 2, 16, 64, dtype=BF16).expand(6, 2, 16, 64)}, ValueError, "no two entries in one place"),
    ({"page_table": torch.zeros(2, 3, dtype=torch.int64)}, TypeError, "page_table must have dtype torch.int32"),
    ({"cu_rows": torch.zeros(3, dtype=torch.int64)}, TypeError, "cu_rows must have dtype torch.int32"),
    ({"lengths": torch.zeros(2, dtype=F32)}, TypeError, "lengths must have dtype torch.int32"),
    ({"cu_rows": torch.zeros(2, dtype=torch.int32)}, ValueError, r"cu_rows must have shape \[3\]"),
    ({"lengths": torch.zeros(3, dtype=torch.int32)}, ValueError, r"lengths must have shape \[2\]"),
    ({"page_table": torch.zeros(2, 0, dtype=torch.int32)}, ValueError, "at least one column"),
    ({"q": torch.zeros(5, 4, 64)}, TypeError, "q must have the dtype of k_pages"),
    ({"q": torch.zeros(5, 4, 32, dtype=BF16)}, ValueError, "q must have shape"),
    ({"q": [1.0]}, TypeError, "q must be a torch.Tensor"),
    ({"out": torch.zeros(5, 4, 64, dtype=F16)}, TypeError, "out must have q's dtype"),
    ({"out": torch.zeros(5, 3, 64, dtype=BF16)}, ValueError, "out must have q's shape"),
    ({"out": torch.zeros(5, 64, 4, dtype=BF16).transpose(1, 2)}, ValueError, "out must be 16-byte aligned"),
    ({"out": torch.zeros(1, 4, 64, dtype=BF16).expand(5, 4, 64)}, ValueError, "out must be 16-byte aligned"),
    ({}, ValueError, "q must be a GPU tensor"),
]


@built
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("change, error, said", BAD_CACHE)
def test_paged_calls_refuse_before_launch(which, change, error, said):
    call = (paged_append_hip, paged_attention_hip)[which]
    arguments = _arguments()[which] | change
    with pytest.raises(error, match=said):
        call(**arguments)


@built
def test_append_and_attention_refuse_their_own():
    append, attention = _arguments()
    for change, error, said in [
            ({"k": torch.zeros(5, 2, 64, dtype=F16)}, TypeError, "k must have the dtype"),
            ({"k": torch.zeros(4, 2, 64, dtype=BF16)}, ValueError, "k must have shape"),
            ({"v": torch.zeros(5, 4, 64, dtype=BF16)}, ValueError, "v must have shape"),
            ({"inv_freq": torch.zeros(32, dtype=torch.float64)}, TypeError, "inv_freq must have dtype"),
            ({"rotary_scale": "1"}, TypeError, "rotary_scale must be a number"),
            ({"v_pages": append["k_pages"]}, ValueError, "must not share memory")]:
        with pytest.raises(error, match=said):
            paged_append_hip(**(append | change))
    for change, error, said in [({"shared_pages": 1.0}, TypeError, "shared_pages must be an integer"),
                                ({"shared_pages": torch.tensor(1)}, TypeError, "shared_pages must be an integer"),
                                ({"shared_pages": 2 ** 70}, ValueError, "shared_pages is out of range"),
                                ({"scale": torch.tensor(1.0)}, TypeError, "scale must be a number"),
                                ({"shared_pages": True}, TypeError, "shared_pages must be an integer"),
                                ({"scale": None, "q": torch.zeros(5, 4, 64, dtype=BF16).requires_grad_()}, RuntimeError,
                                 "has no gradient"),
                                ({"q": torch.nn.Buffer(torch.zeros(5, 4, 64, dtype=BF16))}, ValueError, "GPU tensor")]:
        with pytest.raises(error, match=said):
            paged_attention_hip(**(attention | change))


def _pools():
    """(k_pages, v_pages of [6, 2, 16, 64], whether they lie apart) of one buffer each."""
    def z(*shape):
        return torch.zeros(shape, dtype=BF16)

    yield *z(2, 6, 2, 16, 64).unbind(0), True
    yield *z(6, 2, 2, 16, 64).unbind(1), True          # side by side in a page
    yield *z(6, 2, 2, 16, 64).unbind(2), True          # in a head
    yield *z(6, 2, 16, 2, 64).unbind(3), True          # in a position
    yield *z(6, 2, 16, 128).split(64, 3), True
    yield *(t.transpose(1, 2) for t in z(6, 16, 4, 64).split(2, 2)), True
    pool = z(16, 2, 16, 64)
    yield pool[0:12:2], pool[3:15:2], True             # even pages, odd pages
    yield pool[3:15:2], pool[0:12:2], True
    yield pool[0:12:2], pool[4:16:2], False
    yield pool[:6], pool[5:11], False                  # one page of both
    yield pool[5:11], pool[:6], False
    yield pool[:6], pool[:6], False
    row = z(6 * 2 * 16 * 64 + 8 * 64)
    yield row[:12288].view(6, 2, 16, 64), row[512:].view(6, 2, 16, 64), False  # a position eight further
    wide = z(6, 2, 16, 128)
    yield wide[..., :64], wide[..., 32:96], False      # half of each vector
    yield wide[..., 64:], wide[..., :64], True
    yield pool[:6], pool[:12].view(6, 2, 2, 16, 64)[:, 1], False  # other strides: by their ranges


@built
@pytest.mark.parametrize("k_pages, v_pages, apart", list(_pools()))
def test_pools_that_share_memory_are_refused(k_pages, v_pages, apart):
    append, attention = _arguments()
    for call, arguments in ((paged_append_hip, append), (paged_attention_hip, attention)):
        with pytest.raises(ValueError, match="must be a GPU tensor" if apart else "must not share memory"):
            call(**(arguments | {"k_pages": k_pages, "v_pages": v_pages}))


@built
def test_verify_refuses_before_launch():
    good = {"target_probs": torch.zeros(2, 4, 9), "draft_tokens": torch.zeros(2, 3, dtype=torch.int64),
            "uniforms": torch.zeros(2, 4), "draft_probs": torch.zeros(2, 3, 9),
            "draft_lengths": torch.zeros(2, dtype=torch.int32)}
    for change, error, said in [
            ({"target_probs": torch.zeros(2, 4, 9, dtype=torch.float64)}, TypeError, "target_probs must have dtype"),
            ({"target_probs": torch.zeros(2, 3, 9)}, ValueError, r"target_probs must have shape \[2, 4, 9\]"),
            ({"target_probs": torch.zeros(2, 4, 0)}, ValueError, "at least one entry"),
            ({"draft_tokens": torch.zeros(2, 3, dtype=torch.int32)}, TypeError, "draft_tokens must have dtype"),
            ({"uniforms": torch.zeros(2, 3)}, ValueError, "uniforms must have shape"),
            ({"uniforms": torch.zeros(2, 4, dtype=F16)}, TypeError, "uniforms must have dtype"),
            ({"draft_probs": torch.zeros(2, 3, 9, dtype=BF16)}, TypeError, "draft_probs must have the dtype"),
            ({"draft_probs": torch.zeros(2, 4, 9)}, ValueError, "draft_probs must have shape"),
            ({"draft_lengths": torch.zeros(2, dtype=torch.int64)}, TypeError, "draft_lengths must have dtype"),
            ({"draft_lengths": torch.zeros(3, dtype=torch.int32)}, ValueError, "draft_lengths must have shape"),
            ({}, ValueError, "target_probs must be a GPU tensor")]:
        with pytest.raises(error, match=said):
            verify_drafts_hip(**(good | change))


@built
def test_c_entry_points_refuse_before_launch():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buffer) + 15) & ~15
    null, f = None, ctypes.c_float

    def cache(**change):
        fields = {"k": p, "v": p, "k_page": 2048, "k_head": 1024, "k_position": 64, "v_page": 2048, "v_head": 1024,
                  "v_position": 64, "num_pages": 4, "page_size": 16, "page_table": p, "table_width": 3,
                  "table_stride": 3, "cu_rows": p, "lengths": p, "batch": 2, "kv_heads": 2, "head_dim": 64, "dtype": 2}
        return ctypes.byref(_lib.PagedCache(**(fields | change)))

    row = ctypes.byref(_lib.Rows(p, 128, 64))
    odd = ctypes.byref(_lib.Rows(p + 2, 128, 64))
    slant = ctypes.byref(_lib.Rows(p, 128, 60))

    def append(c, rows=(row, row, row, row), inv=p, rotary=64, scale=1.0, n=1, heads=4):
        return lib.qwen2_paged_append(c, *rows, inv, rotary, 0, f(scale), n, heads, 1, null)

    def attention(c, q=row, out=row, n=1, heads=4, shared=0, scale=0.1, ws=p, nbytes=1 << 20):
        return lib.qwen2_paged_attention(c, q, out, n, heads, shared, f(scale), 1, ws, nbytes, null)

    for call in (append, attention):
        for change, status in [({"dtype": 3}, _lib.STATUS_INVALID_DTYPE), ({"page_size": 8}, 1), ({"page_size": 48}, 1),
                               ({"page_size": 1 << 21}, 1), ({"batch": 0}, 1), ({"kv_heads": 0}, 1),
                               ({"num_pages": 0}, 1), ({"table_width": 0}, 1), ({"k": null}, 1), ({"v": p + 8}, 1),
                               ({"k_head": 1020}, 1), ({"v_page": -8}, 1), ({"cu_rows": null}, 1),
                               ({"lengths": p + 2}, 1), ({"head_dim": 72}, _lib.STATUS_UNSUPPORTED),
                               ({"k_position": 1 << 25}, _lib.STATUS_UNSUPPORTED)]:
            assert call(cache(**change)) == status, (change, lib.w4g64_last_error())
        assert call(null) == 1
        assert call(cache(), n=-1) == 1 and call(cache(), heads=0) == 1
        assert call(cache(), n=0) == _lib.STATUS_OK
    assert append(cache(), rotary=24) == 1 and append(cache(), rotary=80) == 1 and append(cache(), rotary=-16) == 1
    assert append(cache(), scale=math.inf) == 1 and append(cache(), inv=null) == 1
    for bad in (odd, slant, null, ctypes.byref(_lib.Rows(null, 128, 64))):
        assert append(cache(), rows=(row, bad, row, row)) == 1
        assert attention(cache(), q=bad) == 1 and attention(cache(), out=bad) == 1
    assert attention(cache(), heads=5) == 1 and attention(cache(), shared=4) == 1 and attention(cache(), shared=-1) == 1
    assert attention(cache(), scale=math.nan) == 1
    assert attention(cache(table_width=1 << 28)) == _lib.STATUS_UNSUPPORTED
    need = lib.qwen2_paged_attention_workspace_bytes(cache(), 9, 4, 1)
    assert need > 0 and lib.qwen2_paged_attention_workspace_bytes(cache(page_size=8), 9, 4, 1) == 0
    assert attention(cache(), n=9, shared=1, nbytes=need - 1) == _lib.STATUS_WORKSPACE
    assert attention(cache(), n=9, shared=1, ws=null) == _lib.STATUS_WORKSPACE

    def verify(dtype=3, tokens=p, batch=1, drafts=2, vocab=100, ws=p, nbytes=1 << 20, target=p, draft=null):
        return lib.qwen2_verify_drafts(target, 300, 100, draft, 0, 0, dtype, tokens, null, p, p, p, batch, drafts, vocab,
                                       ws, nbytes, null)

    assert verify(dtype=0) == _lib.STATUS_INVALID_DTYPE
    assert verify(vocab=0) == 1 and verify(drafts=-1) == 1 and verify(batch=-1) == 1 and verify(drafts=1 << 16) == 1
    assert verify(target=null) == 1 and verify(tokens=null) == 1 and verify(target=p + 2) == 1 and verify(draft=p + 1) == 1
    assert verify(nbytes=8) == _lib.STATUS_WORKSPACE and verify(ws=null) == _lib.STATUS_WORKSPACE
    assert verify(batch=1 << 31) == _lib.STATUS_UNSUPPORTED
    assert verify(batch=0) == _lib.STATUS_OK


def test_a_missing_host_module_raises(monkeypatch):
    import sys

    from qwen_int4_hip import paged

    if not _lib.library_built():
        pytest.skip("HIP library not built")
    monkeypatch.setattr(paged, "_host", None)
    monkeypatch.delattr(qwen_int4_hip, "_host", raising=False)
    monkeypatch.setitem(sys.modules, "qwen_int4_hip._host", None)
    with pytest.raises(RuntimeError, match="host module is not usable"):
        paged_attention_hip(**_arguments()[1])


# ---------------------------------------------------------------------------
# On the GPU
# ---------------------------------------------------------------------------

class Paged:
    """A pool, its tables and rows: ``rows[b]`` new positions after ``past[b]``
    cached ones, the first ``shared`` pages common.  Pages that nothing names, and
    what lies behind a sequence's end, hold NaN."""

    def __init__(self, rows, past, *, heads=4, kv_heads=2, dim=64, page=16, shared=0, dtype=BF16, token_major=False,
                 spare=3, tail=0, seed=0):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.rows, self.heads, self.kv_heads, self.dim, self.page = rows, heads, kv_heads, dim, page
        self.shared, self.dtype = shared, dtype
        self.lengths_list = [shared * page + n + p for n, p in zip(rows, past)]
        needed = [-(-(n + p) // page) for n, p in zip(rows, past)]
        count = shared + sum(needed) + spare
        order = torch.randperm(count, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((len(rows), max(1, shared + max(needed))), -9, dtype=torch.int32)
        self.used = []  # of each sequence
        for b, n in enumerate(needed):
            own = [order.pop() for _ in range(n)]
            if b == 0:
                first = [order.pop() for _ in range(shared)]
            self.used.append(first + own)
            table[b, :shared + n] = torch.tensor(first + own, dtype=torch.int32)
        self.table = table.cuda()
        self.cu = torch.tensor([0] + rows).cumsum(0).to(torch.int32).cuda()
        self.lengths = torch.tensor(self.lengths_list, dtype=torch.int32).cuda()
        self.total = sum(rows)
        shape = (count, page, kv_heads, dim) if token_major else (count, kv_heads, page, dim)
        self.k_pages, self.v_pages = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2))
        if token_major:
            self.k_pages, self.v_pages = self.k_pages.transpose(1, 2), self.v_pages.transpose(1, 2)
        for b, length in enumerate(self.lengths_list):
            for t in range(0 if b == 0 else shared * page, length, page):
                here = min(page, length - t)
                for cache in (self.k_pages, self.v_pages):
                    cache[self.used[b][t // page], :, :here] = self.randn(kv_heads, here, dim)
        self.q = self.randn(self.total + tail, heads, dim)

    def randn(self, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda").to(self.dtype)

    def cached(self, b, length=None):
        """Keys and values [kv_heads, length, dim] of a sequence, 64 bits."""
        at = torch.arange(self.lengths_list[b] if length is None else length, device="cuda")
        where = torch.tensor(self.used[b] or [0], device="cuda")[at // self.page]
        return tuple(c[where, :, at % self.page].double().transpose(0, 1) for c in (self.k_pages, self.v_pages))

    def attention(self, q=None, **more):
        return paged_attention_hip(self.q if q is None else q, self.k_pages, self.v_pages, self.table, self.cu,
                                   self.lengths, shared_pages=self.shared, **more)

    def reference(self, q=None, scale=None):
        """(attended rows, bound of the fp32 steps' error), 64 bits."""
        q = self.q if q is None else q
        scale = self.dim ** -0.5 if scale is None else scale
        out, slack = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, device="cuda").double()
        group, at = self.heads // self.kv_heads, 0
        for b, n in enumerate(self.rows):
            length = self.lengths_list[b]
            if n and length > 0:
                k, v = (t.repeat_interleave(group, 0) for t in self.cached(b))
                x = q[at:at + n].double().transpose(0, 1)
                first = length - n
                sees = torch.arange(length, device="cuda") <= first + torch.arange(n, device="cuda").view(-1, 1)
                # (what a row does not see is left out of the products: it may be NaN)
                s = torch.where(sees, torch.where(sees.any(0).view(1, 1, -1), (x @ k.transpose(1, 2)) * scale, 0.0),
                                -math.inf)
                w = torch.softmax(s, dim=-1).nan_to_num(0.0) if (first < 0) else torch.softmax(s, dim=-1)
                part = torch.stack([w[:, i, :max(0, first + i + 1)] .unsqueeze(1) @ v[:, :max(0, first + i + 1)]
                                    for i in range(n)], 1).squeeze(2)
                out[at:at + n] = part.transpose(0, 1)
                # a score is a sum of dim products (an error of 2^-24 of their sizes for each, twice for the
                # scale's and the exponential's roundings), a probability is kept to 2^-18, and sums over the
                # keys lose 2^-24 for each block of eight at most: all relative to sum w |v|
                big = (x.abs() @ k.abs().transpose(1, 2)).nan_to_num(0.0).amax() * abs(scale)
                size = torch.stack([w[:, i, :max(0, first + i + 1)].unsqueeze(1) @ v[:, :max(0, first + i + 1)].abs()
                                    for i in range(n)], 1).squeeze(2)
                rel = 2.0 ** -24 * 2 * (self.dim + 8) * big + 2.0 ** -17 + 2.0 ** -24 * (length / 8 + 64)
                slack[at:at + n] = (size * rel).transpose(0, 1)
            at += n
        return out, slack


def _near(got, want, slack):
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * eps  # (a subnormal result's half step)
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    off = torch.where(want.isnan() | (got == want), 0.0, (got - want).abs() - (want.abs() * eps + slack * (1 + eps) + tiny))
    assert float(off.nan_to_num(nan=1e9).amax() if off.numel() else 0) <= 0, float(off.amax())


ATTENTION = [
    # rows, past, and the rest
    ([1], [0], {}),
    ([1], [15], {}),
    ([1], [16], {}),
    ([1], [575], {"heads": 12, "dim": 128}),
    ([1, 1, 1], [3, 200, 31], {"heads": 2, "dim": 128, "dtype": F16}),
    ([1] * 24, list(range(5, 725, 30)), {"heads": 12, "dim": 128}),
    ([2, 0, 5, 1], [0, 7, 33, 64], {"heads": 14, "kv_heads": 2, "dim": 64}),
    ([0, 0, 3], [5, 9, 1], {"heads": 9, "kv_heads": 3, "page": 32}),
    ([5] * 4, [0, 1, 47, 100], {"shared": 9, "heads": 12, "dim": 128}),
    ([1] * 7, [0, 2, 15, 16, 17, 31, 300], {"shared": 1, "heads": 8, "kv_heads": 8, "page": 64, "dtype": F16}),
    ([3, 1, 2], [0, 0, 0], {"shared": 40, "heads": 6, "kv_heads": 1, "dim": 128, "token_major": True}),
    ([70, 1, 33], [0, 400, 5], {"heads": 12, "dim": 128, "page": 32}),
    ([130, 2], [11, 90], {"shared": 3, "heads": 4, "kv_heads": 4, "dtype": F16, "page": 128}),
    ([1] * 70, [b % 40 for b in range(70)], {"shared": 2, "heads": 3, "kv_heads": 1}),
    ([64] * 3, [100, 0, 1], {"shared": 66, "heads": 12, "dim": 128}),
    ([1], [4100], {"heads": 32, "kv_heads": 1, "dim": 128, "page": 1024}),
    ([150, 1, 1, 40], [0, 700, 33, 200], {"heads": 12, "dim": 128}),
    ([90, 30], [64, 7], {"shared": 21, "heads": 16, "kv_heads": 2, "dim": 64, "page": 32, "token_major": True}),
    ([300], [17], {"shared": 1, "heads": 7, "kv_heads": 1, "dtype": F16, "page": 256}),
    ([5] * 40, [3 * b for b in range(40)], {"shared": 130, "heads": 12, "dim": 128}),
]


@gpu
@pytest.mark.parametrize("rows, past, more", ATTENTION)
def test_attention_is_the_formula(rows, past, more):
    p = Paged(rows, past, **more)
    _near(p.attention(), *p.reference())


@gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_scales(scale, dtype):
    p = Paged([4, 1, 2], [30, 100, 0], shared=5, dtype=dtype, dim=128)
    _near(p.attention(scale=scale), *p.reference(scale=scale))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_over_far_apart_scores(dtype):
    """Most keys far below the maximum, so many that they count; then one key that
    outweighs all others, first and last."""
    p = Paged([2, 1], [2000, 900], dtype=dtype, dim=64)
    for spot in (0, 700, 2001):
        k = p.k_pages.clone()
        p.k_pages[p.used[0][spot // 16], :, spot % 16] = 12.0
        p.q[:, :, :] = torch.where(torch.rand(p.q.shape, generator=p.gen, device="cuda") < 0.7, 0.1, 0.9).to(dtype)
        _near(p.attention(), *p.reference())
        p.k_pages.copy_(k)


@gpu
@pytest.mark.parametrize("tail", [0, 3])
@pytest.mark.parametrize("more", [{"shared": 4}, {}, {"page": 128}])
def test_rows_behind_the_last_sequence(tail, more):
    p = Paged([2, 0, 1], [9, 3, 50], tail=tail, heads=6, **more)
    want, slack = p.reference()
    got = p.attention()
    _near(got, want, slack)
    assert not got[p.total:].any()
    out = torch.full_like(p.q, 7.0)
    assert p.attention(out=out) is out
    assert torch.equal(out[:p.total], got[:p.total]) and bool((out[p.total:] == 7.0).all())


@gpu
@pytest.mark.parametrize("shared", [0, 3])
def test_rows_without_a_position_give_zeros(shared):
    p = Paged([3, 2], [20, 1], shared=shared)
    p.lengths_list = [2, 0]  # three rows at -1, 0, 1; two at -2, -1
    p.lengths.copy_(torch.tensor(p.lengths_list))
    p.lengths_list[1] = 0
    got = p.attention()
    _near(got, *p.reference())
    assert not got[0].any() and not got[3:].any() and bool(got[1:3].any())
    p.lengths.fill_(-(2 ** 31))
    assert not p.attention().any()


@gpu
@pytest.mark.parametrize("rows, heads", [([3, 2, 1], 4), ([60, 50, 3], 12)])
def test_sequences_that_end_inside_the_shared_prefix(rows, heads):
    """One of them sees a part of the prefix, one all of it but one position, one more."""
    p = Paged(rows, [0, 0, 9], shared=6, heads=heads, dim=128)
    p.lengths_list = [rows[0] + 7, 95, p.lengths_list[2]]
    p.lengths.copy_(torch.tensor(p.lengths_list))
    _near(p.attention(), *p.reference())


@gpu
def test_lengths_change_between_calls_of_one_shape():
    """The same tables and sizes, every length from one position to the table's end."""
    p = Paged([2], [126], heads=12, dim=128)
    whole = p.lengths_list[0]
    for length in list(range(1, 70)) + [whole - 1, whole]:
        p.lengths_list = [length]
        p.lengths.fill_(length)
        _near(p.attention(), *p.reference())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shared", [0, 2])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_a_row_does_not_see_takes_no_part(dtype, shared, bad):
    """The fourth of six new positions holds values (then keys) that are not finite:
    the rows before it are unmoved, those from it on are not finite."""
    p = Paged([6, 1], [21, 70], shared=shared, dtype=dtype, heads=6, dim=128)
    want, slack = p.reference()
    spot = shared * 16 + 21 + 3
    page, place = p.used[0][spot // 16], spot % 16
    for cache in (p.v_pages, p.k_pages):
        kept = cache[page, :, place].clone()
        cache[page, :, place] = bad
        got = p.attention()
        _near(got[:3], want[:3], slack[:3])
        _near(got[6:], want[6:], slack[6:])
        if cache is p.v_pages:
            assert bool((got[3:6].isnan() if math.isnan(bad) else got[3:6] == bad).all())
        elif math.isnan(bad):
            assert bool(got[3:6].isnan().all())
        cache[page, :, place] = kept
    # one visible value only, in a long context: its dimension alone
    p.v_pages[p.used[1][-1], 0, 0, 5] = bad
    changed = p.attention()
    touched = torch.zeros_like(changed, dtype=torch.bool)
    touched[6, :3, 5] = True
    assert not changed[touched].isfinite().any()
    _near(torch.where(touched, 0, changed), torch.where(touched, 0.0, want), slack)


@gpu
@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (F16, 64), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("shared", [0, 9])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite_among_many_rows(dtype, dim, shared, bad):
    """Sequences of 40, one and 30 rows, 6 query heads each: whole values at one new
    position, and one element that all rows see, in the prefix or at the start."""
    p = Paged([40, 1, 30], [21, 70, 3], shared=shared, dtype=dtype, heads=12, dim=dim)
    want, slack = p.reference()
    spot = shared * 16 + 21 + 17
    page, place = p.used[0][spot // 16], spot % 16
    kept = p.v_pages[page, :, place].clone()
    p.v_pages[page, :, place] = bad
    got = p.attention()
    _near(got[:17], want[:17], slack[:17])
    _near(got[40:], want[40:], slack[40:])
    assert bool((got[17:40].isnan() if math.isnan(bad) else got[17:40] == bad).all())
    p.v_pages[page, :, place] = kept
    p.v_pages[p.used[0][0], 1, 3, 7] = bad  # (key/value head 1: query heads 6 ..)
    got = p.attention()
    touched = torch.zeros_like(got, dtype=torch.bool)
    touched[:71 if shared else 40, 6:, 7] = True
    seen = got[touched]
    assert bool((seen.isnan() if math.isnan(bad) else seen == bad).all())
    _near(torch.where(touched, 0, got), torch.where(touched, 0.0, want), slack)
    p.v_pages[p.used[0][0], 1, 4, 7] = -bad  # (another key's: their sum has no value)
    assert bool(p.attention()[touched].isnan().all())


@gpu
@pytest.mark.parametrize("shared", [0, 2])
def test_pages_that_are_not_there_give_nan(shared):
    p = Paged([3, 2, 1], [40, 2, 100], shared=shared, heads=6)
    want, slack = p.reference()
    for value in (-1, p.k_pages.shape[0], 2 ** 31 - 1, -(2 ** 31)):
        table = p.table.clone()
        table[0, shared + 2] = value  # (the rows at 40, 41 and 42 all sit in the third own page)
        got = paged_attention_hip(p.q, p.k_pages, p.v_pages, table, p.cu, p.lengths, shared_pages=shared)
        assert bool(got[:3].isnan().all())
        _near(got[3:], want[3:], slack[3:])
        if shared:
            table = p.table.clone()
            table[0, 0] = value
            assert bool(paged_attention_hip(p.q, p.k_pages, p.v_pages, table, p.cu, p.lengths,
                                            shared_pages=shared).isnan().all())
    # a bad page that only the last of three rows reaches
    q = Paged([3], [30], heads=2)
    want, slack = q.reference()
    q.table[0, 2] = -1
    got = q.attention()
    assert bool(got[2].isnan().all())
    _near(got[:2], want[:2], slack[:2])
    # a length past the table: the rows that reach there, in a call with and without own pages
    q = Paged([2], [13], heads=2)
    for cache in (q.k_pages, q.v_pages):
        cache[q.used[0][0], :, 15] = 1.0
    q.lengths.fill_(17)  # rows at 15, 16 of a table of 16
    got = q.attention()
    assert bool(got[1].isnan().all()) and bool(got[0].isfinite().all())
    got = paged_attention_hip(q.q, q.k_pages, q.v_pages, q.table, q.cu, q.lengths, shared_pages=1)
    assert bool(got[1].isnan().all()) and bool(got[0].isfinite().all())
    q.lengths.fill_(2 ** 31 - 1)
    assert bool(q.attention().isnan().all())


@gpu
@pytest.mark.parametrize("shared", [0, 2])
def test_pages_that_are_not_there_among_many_rows(shared):
    """Sixty rows of six heads at own positions 40 .. 99; the page of 80 .. 95, then one
    of the prefix, then the table's end."""
    p = Paged([60, 45], [40, 2], shared=shared, heads=12, dim=128)
    want, slack = p.reference()
    table = p.table.clone()
    table[0, shared + 5] = -1
    got = paged_attention_hip(p.q, p.k_pages, p.v_pages, table, p.cu, p.lengths, shared_pages=shared)
    assert bool(got[40:60].isnan().all())
    _near(got[:40], want[:40], slack[:40])
    _near(got[60:], want[60:], slack[60:])
    if shared:
        table = p.table.clone()
        table[0, 1] = p.k_pages.shape[0]
        assert bool(paged_attention_hip(p.q, p.k_pages, p.v_pages, table, p.cu, p.lengths,
                                        shared_pages=shared).isnan().all())
    reach = p.table.shape[1] * 16
    for cache in (p.k_pages, p.v_pages):  # (all that the table names is written)
        cache[p.used[0]] = cache[p.used[0]].nan_to_num(0.5)
    lengths = p.lengths.clone()
    lengths[0] = reach + 10
    got = paged_attention_hip(p.q, p.k_pages, p.v_pages, p.table, p.cu, lengths, shared_pages=shared)
    assert bool(got[50:60].isnan().all()) and bool(got[:50].isfinite().all())
    _near(got[60:], want[60:], slack[60:])


@gpu
@pytest.mark.parametrize("values", [[-7, 90, 2, -1], [5, 5, 5, 5], [0, 2 ** 31 - 1, -(2 ** 31), 4]])
def test_row_bounds_that_fall_or_lead_out_stay_in_the_buffers(values):
    """What cu_rows should not hold: nothing is promised but that nothing faults
    and that rows behind the last bound keep what they hold."""
    p = Paged([2, 1, 1], [3, 40, 9], shared=2)
    p.cu.copy_(torch.tensor(values, dtype=torch.int64).to(torch.int32))
    out = torch.full_like(p.q, 7.0)
    p.attention(out=out)
    p.attention()
    paged_append_hip(p.q, p.randn(4, 2, 64), p.randn(4, 2, 64), p.k_pages, p.v_pages, p.table, p.cu, p.lengths, None)
    torch.cuda.synchronize()


@gpu
def test_attention_reads_strided_and_unaligned_rows():
    p = Paged([3, 1], [20, 5], heads=4, dim=64, shared=1)
    want = p.attention()
    wide = torch.zeros(4, 12, 64, dtype=BF16, device="cuda")
    wide[:, 3:11:2] = p.q
    assert torch.equal(p.attention(q=wide[:, 3:11:2]), want)
    odd = torch.zeros(4 * 4 * 64 + 3, dtype=BF16, device="cuda")[3:].view(4, 4, 64)
    odd.copy_(p.q)
    assert torch.equal(p.attention(q=odd), want)
    assert torch.equal(p.attention(q=p.q.transpose(0, 1).contiguous().transpose(0, 1)), want)
    out = torch.zeros(4, 4, 128, dtype=BF16, device="cuda")[..., 64:]
    assert torch.equal(p.attention(out=out), want)
    table = torch.full((2, 2 * p.table.shape[1]), -1, dtype=torch.int32, device="cuda")
    table[:, ::2] = p.table
    for t in (table[:, ::2], torch.cat((p.table, p.table), 1)[:, :p.table.shape[1]]):
        assert torch.equal(paged_attention_hip(p.q, p.k_pages, p.v_pages, t, p.cu, p.lengths, shared_pages=1), want)
    # one pool with keys and values side by side
    both = torch.zeros(p.k_pages.shape[0], 2, 2, 16, 64, dtype=BF16, device="cuda")
    both[:, 0], both[:, 1] = p.k_pages, p.v_pages
    assert torch.equal(paged_attention_hip(p.q, both[:, 0], both[:, 1], p.table, p.cu, p.lengths, shared_pages=1), want)
    with pytest.raises(ValueError, match="share no memory"):
        p.attention(out=p.q)
    with pytest.raises(ValueError, match="must not share memory"):
        paged_attention_hip(p.q, p.k_pages, p.k_pages, p.table, p.cu, p.lengths)


@gpu
def test_attention_of_nothing():
    p = Paged([0, 0], [5, 3])
    assert p.attention().shape == (0, 4, 64)
    none = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    got = paged_attention_hip(p.randn(3, 4, 64), p.k_pages, p.v_pages, none, none.new_zeros(1), none.new_zeros(0))
    assert got.shape == (3, 4, 64) and not got.any()


@gpu
def test_pages_past_32_bit_offsets():
    """A pool of more than 2^31 elements, its last pages in use."""
    page, kv_heads, dim, count = 64, 2, 128, 131080 + 16
    pools = [torch.empty(count, kv_heads, page, dim, dtype=BF16, device="cuda") for _ in range(2)]
    used = [count - 1, count - 7, 3]
    gen = torch.Generator(device="cuda").manual_seed(3)
    small = [torch.randn(3, kv_heads, page, dim, generator=gen, device="cuda").to(BF16) for _ in range(2)]
    for pool, part in zip(pools, small):
        pool[used] = part
    table = torch.tensor([used], dtype=torch.int32, device="cuda")
    cu, lengths = torch.tensor([0, 2], dtype=torch.int32, device="cuda"), torch.tensor([150], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(2, h, dim, generator=gen, device="cuda").to(BF16) for h in (12, 2, 2))
    ids = torch.arange(3, dtype=torch.int32, device="cuda").view(1, 3)
    inv = torch.rand(64, device="cuda")
    a = paged_append_hip(q, k, v, *pools, table, cu, lengths, inv)
    b = paged_append_hip(q, k, v, *small, ids, cu, lengths, inv)
    assert torch.equal(a, b)
    for pool, part in zip(pools, small):
        assert torch.equal(pool[used], part)
    for shared in (0, 1):
        assert torch.equal(paged_attention_hip(a, *pools, table, cu, lengths, shared_pages=shared),
                           paged_attention_hip(a, *small, ids, cu, lengths, shared_pages=shared))


# ---- append ----

def _turned(x, positions, inv_freq, interleaved, scale):
    """Rows rotated in 64 bits, and sum |products| for the fp32 steps' error."""
    x = x.double()
    if inv_freq is None or not inv_freq.numel():
        return x, torch.zeros_like(x)
    rotary = 2 * inv_freq.numel()
    angle = (positions.double().view(-1, 1) * inv_freq.double()).view(x.shape[0], 1, -1)
    cos, sin = angle.cos() * scale, angle.sin() * scale
    one, two = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:rotary])
    a, b = one * cos - two * sin, two * cos + one * sin
    sizes = (one.abs() + two.abs()) * abs(scale)
    out, size = x.clone(), torch.zeros_like(x)
    if interleaved:
        out[..., 0:rotary:2], out[..., 1:rotary:2] = a, b
        size[..., 0:rotary:2], size[..., 1:rotary:2] = sizes, sizes
    else:
        out[..., :rotary // 2], out[..., rotary // 2:rotary] = a, b
        size[..., :rotary // 2], size[..., rotary // 2:rotary] = sizes, sizes
    # the angle left after whole turns to 2^-24 of half a turn (pi 2^-24 < 2^-22), sine and cosine to two
    # units, a product and a sum: below 2^-20 of the sizes
    return out, size * 2.0 ** -20


APPEND = [
    # rows, past, heads, kv_heads, dim, rotary, page, interleaved, dtype, token_major
    ([1], [0], 1, 1, 16, 16, 16, False, BF16, False),
    ([1], [575], 12, 2, 128, 128, 16, False, BF16, False),
    ([5, 0, 17, 1], [3, 9, 30, 15], 12, 2, 128, 128, 16, False, BF16, False),
    ([5, 0, 17, 1], [3, 9, 30, 15], 9, 3, 96, 32, 32, True, F16, True),
    ([1] * 70, list(range(70)), 4, 4, 64, 64, 64, True, BF16, False),
    ([300, 2], [1, 7], 14, 2, 64, 16, 128, False, F16, False),
    ([2, 3], [40, 0], 6, 6, 256, 256, 16, True, BF16, True),
    ([2, 3], [40, 0], 5, 1, 256, 224, 16, False, F16, False),
    ([3], [14], 3, 1, 48, 0, 16, False, BF16, False),
]


@gpu
@pytest.mark.parametrize("rows, past, heads, kv_heads, dim, rotary, page, interleaved, dtype, token_major", APPEND)
def test_append_is_the_formula(rows, past, heads, kv_heads, dim, rotary, page, interleaved, dtype, token_major):
    p = Paged(rows, past, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, token_major=token_major)
    scale = 1.0 if interleaved else 1.3
    inv = None if not rotary else 10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=F32) / rotary)
    qkv = p.randn(p.total, heads + 2 * kv_heads, dim)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), dim=1)
    before = [c.clone() for c in (p.k_pages, p.v_pages)]
    got = paged_append_hip(q, k, v, p.k_pages, p.v_pages, p.table, p.cu, p.lengths, inv, interleaved=interleaved,
                           rotary_scale=scale)
    assert got.is_contiguous()
    positions = torch.cat([torch.arange(n - r, n) for n, r in zip(p.lengths_list, rows)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows)).cuda()
    where = p.table.long()[seq, positions // page]
    _near(got, *_turned(q, positions, inv, interleaved, scale))
    _near(p.k_pages[where, :, positions % page], *_turned(k, positions, inv, interleaved, scale))
    assert torch.equal(p.v_pages[where, :, positions % page], v)
    for cache, old in zip((p.k_pages, p.v_pages), before):  # and nothing else
        cache, old = cache.clone(), old
        cache[where, :, positions % page] = 0
        old[where, :, positions % page] = 0
        assert torch.equal(cache.contiguous().view(torch.int16), old.contiguous().view(torch.int16))
    # in place, and into strided rows
    spare = qkv.clone()
    q2 = spare[:, :heads]
    assert paged_append_hip(q2, k, v, p.k_pages, p.v_pages, p.table, p.cu, p.lengths, inv, interleaved=interleaved,
                            rotary_scale=scale, out=q2) is q2
    assert torch.equal(q2, got) and torch.equal(spare[:, heads:], qkv[:, heads:])


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_far_positions(interleaved):
    """Positions to 16 million: the angle's whole turns come off in 64 bits."""
    page, dim = 1 << 18, 64
    k_pages, v_pages = (torch.zeros(1, 1, page, dim, dtype=F16, device="cuda") for _ in range(2))
    table = torch.zeros(1, 64, dtype=torch.int32, device="cuda")
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=F32) / dim)
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(9, h, dim, generator=gen, device="cuda").to(F16) for h in (3, 1, 1))
    cu = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    for length in (1_000_003, 64 * page):
        lengths = torch.tensor([length], dtype=torch.int32, device="cuda")
        got = paged_append_hip(q, k, v, k_pages, v_pages, table, cu, lengths, inv, interleaved=interleaved)
        positions = torch.arange(length - 9, length, device="cuda")
        _near(got, *_turned(q, positions, inv, interleaved, 1.0))
        _near(k_pages[0, :, positions % page].transpose(0, 1), *_turned(k, positions, inv, interleaved, 1.0))


@gpu
def test_append_leaves_what_it_may_not_write():
    p = Paged([2, 3, 1], [30, 3, 0], heads=4, tail=2)
    k, v = p.randn(8, 2, 64), p.randn(8, 2, 64)
    inv = torch.rand(32, device="cuda")
    for cache in (p.k_pages, p.v_pages):
        cache.fill_(5.0)
    table = p.table.clone()
    table[0, 1] = -1               # position 30 is nowhere, 31 neither
    lengths = p.lengths.clone()
    lengths[1] = 2                 # three rows at -1, 0, 1
    lengths[2] = 10 ** 9           # past its table
    out = torch.full((8, 4, 64), 7.0, dtype=BF16, device="cuda")
    paged_append_hip(p.q, k, v, p.k_pages, p.v_pages, table, p.cu, lengths, inv, out=out)
    positions = torch.tensor([30, 31, -1, 0, 1, 10 ** 9 - 1], device="cuda")
    _near(out[:6], *_turned(p.q[:6], positions, inv, False, 1.0))
    assert bool((out[6:] == 7.0).all())
    spots = (p.v_pages != 5.0).any(-1).any(1)  # [pages, places]
    want = torch.zeros_like(spots)
    want[p.used[1][0], :2] = True
    assert torch.equal(spots, want) and torch.equal(p.v_pages[p.used[1][0], :, :2].transpose(0, 1), v[3:5])
    fresh = paged_append_hip(p.q, k, v, p.k_pages, p.v_pages, table, p.cu, lengths, inv)
    assert torch.equal(fresh[:6], out[:6]) and not fresh[6:].any()


@gpu
def test_append_copies_rows_it_cannot_read_in_place():
    p = Paged([3, 2], [7, 0], heads=4)
    k, v, inv = p.randn(5, 2, 64), p.randn(5, 2, 64), torch.rand(32, device="cuda")
    got = paged_append_hip(p.q, k, v, p.k_pages, p.v_pages, p.table, p.cu, p.lengths, inv)
    want = p.k_pages.clone(), p.v_pages.clone()

    def odd(t):
        moved = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return moved.copy_(t)

    again = paged_append_hip(odd(p.q), odd(k), v.transpose(1, 2).contiguous().transpose(1, 2), p.k_pages, p.v_pages,
                             p.table, p.cu, p.lengths, odd(inv))
    assert torch.equal(again, got)
    for cache, old in zip((p.k_pages, p.v_pages), want):
        assert torch.equal(cache.view(torch.int16), old.view(torch.int16))
    base = torch.zeros(6 * 4, 64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="out must be q itself"):
        paged_append_hip(base[:20].view(5, 4, 64), k, v, p.k_pages, p.v_pages, p.table, p.cu, p.lengths, inv,
                         out=base[4:].view(5, 4, 64))
    one = torch.zeros(5, 2, 64, dtype=BF16, device="cuda")  # queries and keys of one tensor
    assert torch.equal(paged_append_hip(one, one, one, p.k_pages, p.v_pages, p.table, p.cu, p.lengths, inv), one)
    with pytest.raises(ValueError, match="must not share its rows"):
        paged_append_hip(one, one, one, p.k_pages, p.v_pages, p.table, p.cu, p.lengths, inv, out=one)
    with pytest.raises(ValueError, match="the cache must not share memory"):
        paged_append_hip(p.q, p.k_pages[:5, :, 0], v, p.k_pages, p.v_pages, p.table, p.cu, p.lengths, inv)


# ---- verify ----

def _verified(target, tokens, uniforms, draft, lengths=None):
    target, uniforms = target.double().cpu(), uniforms.double().cpu()
    draft = None if draft is None else draft.double().cpu()
    batch, drafts = tokens.shape
    out, counts = torch.full((batch, drafts + 1), -1), torch.zeros(batch, dtype=torch.int32)
    below_one = 1.0 - 2.0 ** -24
    for b in range(batch):
        count = drafts if lengths is None else min(max(int(lengths[b]), 0), drafts)
        n = 0
        while n < count:
            x = int(tokens[b, n])
            if not 0 <= x < target.shape[2]:
                break
            q = 1.0 if draft is None else float(draft[b, n, x])
            if not float(uniforms[b, n]) * q < float(target[b, n, x]):
                break
            out[b, n] = x
            n += 1
        weight = target[b, n].clone()
        if n < count:
            if draft is not None:
                weight -= draft[b, n]
            elif 0 <= int(tokens[b, n]) < weight.numel():
                weight[int(tokens[b, n])] -= 1.0
        weight = weight.clamp_min(0)
        if float(weight.sum()) == 0.0:
            weight = target[b, n].clamp_min(0)
        run = weight.cumsum(0)
        u = min(max(float(uniforms[b, drafts]), 0.0), below_one)
        if 0 < float(run[-1]) < math.inf and uniforms[b, drafts] == uniforms[b, drafts]:
            out[b, n] = int(torch.searchsorted(run, u * run[-1], right=True))
        counts[b] = n
    return out, counts


def _same(got, want):
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.int32
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("batch, drafts, vocab", [(1, 1, 1), (1, 4, 151936), (3, 2, 4096), (2, 7, 4097), (17, 3, 5001),
                                                  (5, 0, 300), (2, 130, 77), (66, 1, 16), (2, 2, 32768), (2, 3, 32769), (257, 1, 40001)])
@pytest.mark.parametrize("copied", [False, True])
def test_verify_is_the_formula(dtype, batch, drafts, vocab, copied):
    gen = torch.Generator(device="cuda").manual_seed(batch * 1000 + drafts)
    logits = 2 * torch.randn(batch, drafts + 1, vocab, generator=gen, device="cuda")
    target = torch.softmax(logits, -1).to(dtype)
    noise = torch.randn(batch, drafts, vocab, generator=gen, device="cuda")
    draft = torch.softmax(logits[:, :drafts] + (0.05 if drafts > 50 else 0.7) * noise, -1)
    tokens = torch.multinomial(draft.reshape(-1, vocab), 1, generator=gen).view(batch, drafts) if drafts else \
        torch.zeros(batch, 0, dtype=torch.int64, device="cuda")
    draft = None if copied else draft.to(dtype)
    uniforms = torch.rand(batch, drafts + 1, generator=gen, device="cuda")
    lengths = torch.arange(batch, dtype=torch.int32, device="cuda") % (drafts + 3) - 1
    for n in (None, lengths):
        _same(verify_drafts_hip(target, tokens, uniforms, draft_probs=draft, draft_lengths=n),
              _verified(target, tokens, uniforms, draft, n))


@gpu
def test_verify_on_borders():
    """Probabilities in eighths, uniforms on the borders: equality does not pass."""
    eighth = torch.tensor([1, 0, 3, 2, 0, 1, 1, 0], device="cuda") / 8
    drawn = torch.tensor([2, 1, 1, 1, 1, 1, 1, 0], device="cuda") / 8
    for i in range(8):
        for k in range(8):
            target, draft = eighth.expand(1, 2, 8).contiguous(), drawn.expand(1, 1, 8).contiguous()
            tokens = torch.tensor([[k]], device="cuda")
            uniforms = torch.tensor([[i / 8, i / 8]], device="cuda")
            for q in (draft, None):
                _same(verify_drafts_hip(target, tokens, uniforms, draft_probs=q), _verified(target, tokens, uniforms, q))


@gpu
@pytest.mark.parametrize("vocab", [3, 5000, 40000])
def test_verify_falls_back_to_the_target(vocab):
    """A draft that is nowhere below the target, refused: drawn from the target."""
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    target = torch.softmax(torch.randn(4, 2, vocab, generator=gen, device="cuda"), -1)
    draft = 1.25 * target[:, :1]
    tokens = torch.randint(0, vocab, (4, 1), generator=gen, device="cuda")
    uniforms = torch.rand(4, 2, generator=gen, device="cuda")
    uniforms[:, 0] = 0.9  # (past 0.8: refused)
    got = verify_drafts_hip(target, tokens, uniforms, draft_probs=draft)
    _same(got, _verified(target, tokens, uniforms, draft))
    assert got[1].tolist() == [0] * 4 and int(got[0][:, 0].min()) >= 0


@gpu
def test_verify_edges():
    third = torch.full((1, 3, 9), 1 / 9, device="cuda")
    tokens = torch.tensor([[4, 2]], device="cuda")
    zero = torch.zeros(1, 3, device="cuda")
    # a draft equal to the target, refused by a uniform of one: the target alone is left
    one = torch.tensor([[1.0, 0.0, 0.99]], device="cuda")
    _same(verify_drafts_hip(third, tokens, one, draft_probs=third[:, :2]), _verified(third, tokens, one, third[:, :2]))
    # uniforms outside [0, 1): the last entry, the first; not a number: no choice
    for u, want in ((1.0, 8), (7.0, 8), (-1.0, 0), (math.nan, -1)):
        got = verify_drafts_hip(third[:, :1], tokens[:, :0], torch.full((1, 1), u, device="cuda"))
        assert got[0].tolist() == [[want]] and got[1].tolist() == [0]
    # ids outside the vocabulary do not stand
    for bad in (-1, 9, 2 ** 62, -(2 ** 62)):
        for draft in (None, third[:, :2]):
            ids = torch.tensor([[4, bad]], device="cuda")
            u = torch.tensor([[0.0, 0.0, 0.6]], device="cuda")
            got = verify_drafts_hip(third, ids, u, draft_probs=draft)
            assert got[1].tolist() == [1] and got[0][0, 0] == 4 and got[0][0, 2] == -1
            # one-hot at no entry: the target; the draft equals the target: the target
            assert int(got[0][0, 1]) == 5
    # weights that add up to nothing, to infinity, to no number
    for value in (0.0, math.inf, math.nan):
        bad = third.clone()
        bad[0, 0] = value
        got = verify_drafts_hip(bad, torch.tensor([[9, 9]], device="cuda"), zero)
        assert got[0].tolist() == [[-1, -1, -1]] and got[1].tolist() == [0]
    # negative entries weigh nothing
    low = third.clone()
    low[0, 0, :8] = -0.5
    got = verify_drafts_hip(low, torch.tensor([[9, 9]], device="cuda"), zero)
    assert got[0].tolist() == [[8, -1, -1]]
    empty = verify_drafts_hip(third[:0], tokens[:0], zero[:0], draft_probs=third[:0, :2])
    assert empty[0].shape == (0, 3) and empty[1].shape == (0,)


@gpu
def test_verify_reads_strided_probabilities():
    gen = torch.Generator(device="cuda").manual_seed(9)
    base = torch.softmax(torch.randn(5, 6, 1003, generator=gen, device="cuda"), -1)
    tokens = torch.randint(0, 1001, (5, 2), generator=gen, device="cuda")
    uniforms = torch.rand(5, 3, generator=gen, device="cuda")
    views = [(base[:, :3, :1001], base[:, 3:5, 1:1002]),
             (base.transpose(1, 2).contiguous().transpose(1, 2)[:, :3, :1001], base[:, 3:5, 2:]),
             (base[:, :3, 2:].to(BF16)[..., 1:], base[:, 3:5, 3:].to(BF16)),
             (base[:1, :3, 3:].expand(5, 3, 1000), base[:1, 3:4, 3:].expand(5, 2, 1000))]
    for target, draft in views:
        draft = draft[..., :target.shape[2]]
        target = target[..., :draft.shape[2]]
        ids = tokens.clamp_max(target.shape[2] - 1)
        want = _verified(target, ids, uniforms, draft)
        _same(verify_drafts_hip(target, ids, uniforms, draft_probs=draft), want)
        _same(verify_drafts_hip(target, ids.t().contiguous().t(), uniforms.repeat(1, 2)[:, :3], draft_probs=draft), want)


# ---- together, captured, on other streams ----

class Step:
    """One speculative step of a one-layer model with random weights: rows from
    token embeddings, append, attention, probabilities by a head, verification."""

    def __init__(self, batch=3, drafts=3, shared=4, dtype=BF16):
        heads, kv_heads, dim, vocab = 6, 2, 64, 500
        self.p = Paged([drafts + 1] * batch, [5, 60, 17][:batch], heads=heads, kv_heads=kv_heads, dim=dim, shared=shared,
                       dtype=dtype)
        gen = self.p.gen
        self.drafts, self.batch, self.vocab = drafts, batch, vocab
        self.embed = torch.randn(vocab, heads + 2 * kv_heads, dim, generator=gen, device="cuda").to(dtype)
        self.head = torch.randn(heads * dim, vocab, generator=gen, device="cuda") / 8
        self.inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=F32) / dim)
        self.tokens = torch.randint(0, vocab, (batch, drafts + 1), generator=gen, device="cuda")
        self.draft = torch.softmax(torch.randn(batch, drafts, vocab, generator=gen, device="cuda"), -1)
        self.uniforms = torch.rand(batch, drafts + 1, generator=gen, device="cuda")

    def __call__(self):
        p = self.p
        q, k, v = self.embed[self.tokens.view(-1)].split((p.heads, p.kv_heads, p.kv_heads), 1)
        rotated = paged_append_hip(q, k, v, p.k_pages, p.v_pages, p.table, p.cu, p.lengths, self.inv)
        attended = p.attention(q=rotated)
        logits = attended.float().flatten(1) @ self.head
        target = torch.softmax(logits, -1).view(self.batch, self.drafts + 1, self.vocab)
        tokens, accepted = verify_drafts_hip(target, self.tokens[:, 1:], self.uniforms, draft_probs=self.draft)
        return rotated, attended, target, tokens, accepted

    def fresh(self, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.tokens.copy_(torch.randint(0, self.vocab, self.tokens.shape, generator=gen, device="cuda"))
        self.uniforms.copy_(torch.rand(self.uniforms.shape, generator=gen, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_speculative_step(dtype):
    """Three steps, the accepted positions kept, against 64 bits at every joint."""
    s = Step(dtype=dtype)
    p = s.p
    for turn in range(3):
        s.fresh(turn)
        rotated, attended, target, tokens, accepted = s()
        q = s.embed[s.tokens.view(-1)][:, :p.heads]
        positions = torch.cat([torch.arange(n - r, n) for n, r in zip(p.lengths_list, p.rows)]).cuda()
        _near(rotated, *_turned(q, positions, s.inv, False, 1.0))
        _near(attended, *p.reference(q=rotated))
        want = _verified(target, s.tokens[:, 1:], s.uniforms, s.draft)
        _same((tokens, accepted), want)
        # the next step's rows follow the accepted ones (and the new token's row is the first of them)
        stay = [n - s.drafts + int(a) for n, a in zip(p.lengths_list, accepted.tolist())]
        held = [len(u) * p.page for u in p.used]
        p.lengths_list = [min(n, h - s.drafts - 1) + s.drafts for n, h in zip(stay, held)]
        p.lengths.copy_(torch.tensor(p.lengths_list))


@gpu
def test_a_captured_step_follows_its_buffers():
    """One capture, replayed over other tokens and lengths, with eager calls between."""
    s, other = Step(), Step(batch=2, drafts=1, shared=0)
    p = s.p
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s()
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = s()
    with torch.cuda.graph(second, stream=side):  # (its workspaces are its own)
        more = other()
    lengths = p.lengths.clone()
    for turn in range(4):
        s.fresh(10 + turn)
        other.fresh(20 + turn)
        p.lengths.copy_(lengths - turn)
        p.cu.copy_(torch.tensor([0, 4, 8, 12]) if turn != 2 else torch.tensor([0, 4, 4, 8]))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        second.replay()  # (on another stream than the first, at the same time)
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got], [t.clone() for t in more]
        caches = p.k_pages.clone(), p.v_pages.clone()
        for pair in zip(replayed[0], s()):
            assert torch.equal(*(t.view(torch.int16) if t.dtype == BF16 else t for t in pair)), turn
        for pair in zip(replayed[1], other()):
            assert torch.equal(*pair), turn
        for cache, old in zip((p.k_pages, p.v_pages), caches):
            assert torch.equal(cache.view(torch.int16), old.view(torch.int16))


@gpu
def test_calls_on_several_streams_and_modes():
    p = Paged([2, 1, 3], [100, 700, 30], shared=6, heads=12, dim=128)
    want = p.attention()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for stream in streams:
        with torch.cuda.stream(stream):
            got += [p.attention() for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    with torch.inference_mode():
        assert torch.equal(p.attention(), want)
    with torch.device("cuda"):  # a default device
        assert torch.equal(p.attention(), want)
    q = p.q.clone().requires_grad_()
    with torch.no_grad():
        assert torch.equal(p.attention(q=q), want)
    with pytest.raises(RuntimeError, match="has no gradient"):
        p.attention(q=q)
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(RuntimeError, match="dispatch mode"):
        p.attention()
    with pytest.raises(RuntimeError, match="function transform"):
        torch.func.vmap(lambda x: p.attention(q=x))(p.q.unsqueeze(0))
    import torch.autograd.forward_ad as fwAD

    with fwAD.dual_level(), pytest.raises(RuntimeError, match="has no gradient"):
        p.attention(q=fwAD.make_dual(p.q, torch.ones_like(p.q)))
    version = p.k_pages._version
    paged_append_hip(p.q, p.randn(6, 2, 128), p.randn(6, 2, 128), p.k_pages, p.v_pages, p.table, p.cu, p.lengths, None)
    assert p.k_pages._version > version


# ---- what the device's own bounds hold back ----

class Guarded:
    """A buffer filled with one value, of which ``t`` is the middle."""

    def __init__(self, *shape, dtype=BF16, value=9.0, margin=4096):
        count = math.prod(shape)
        self.all = torch.full((count + 2 * margin,), value, dtype=dtype, device="cuda")
        self.t, self.value, self.margin = self.all[margin:margin + count].view(shape), value, margin

    def kept(self):
        return bool((self.all[:self.margin] == self.value).all() and (self.all[-self.margin:] == self.value).all())


def _c_cache(p, table, cu, lengths):
    k, v = p.k_pages, p.v_pages
    return _lib.PagedCache(k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], k.shape[0], k.shape[2],
                           table.data_ptr(), table.shape[1], table.stride(0), cu.data_ptr(), lengths.data_ptr(),
                           table.shape[0], k.shape[1], k.shape[3], {F16: 1, BF16: 2}[k.dtype])


def _c_attention(p, out, *, cu, zero_rest, table=None, lengths=None, shared=0):
    """The C entry point, so that rows behind the last sequence can be zeroed in a buffer of the test's."""
    lib = _lib.load()
    cache = _c_cache(p, p.table if table is None else table, cu, p.lengths if lengths is None else lengths)
    rows = [_lib.Rows(t.data_ptr(), t.stride(0), t.stride(1)) for t in (p.q, out)]
    need = lib.qwen2_paged_attention_workspace_bytes(ctypes.byref(cache), p.q.shape[0], p.heads, shared)
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    _lib.check(lib.qwen2_paged_attention(ctypes.byref(cache), *map(ctypes.byref, rows), p.q.shape[0], p.heads, shared,
                                         p.dim ** -0.5, zero_rest, workspace.data_ptr(), need, _stream()))
    return need


def _stream():
    return torch.cuda.current_stream().cuda_stream


@gpu
@pytest.mark.parametrize("last", [2 ** 31 - 1, 2 ** 31 - 2, 5, 3, -1, -(2 ** 31)])
@pytest.mark.parametrize("zero_rest", [0, 1])
def test_a_last_bound_outside_the_rows(last, zero_rest):
    """One split (the call's own stores see to the rows behind the last sequence), three
    rows: whatever the last bound is, only rows behind it (all, where it is negative)
    are zeroed, and nothing outside them is written."""
    p = Paged([2, 1], [3, 40], heads=4)
    cu = torch.tensor([0, 2, last], dtype=torch.int64).to(torch.int32).to(p.q.device)
    out = Guarded(3, 4, 64)
    assert _c_attention(p, out.t, cu=cu, zero_rest=zero_rest) == 0  # (no workspace: one split)
    assert out.kept()
    want, slack = p.reference()
    if last >= 3:
        _near(out.t, want, slack)
    elif zero_rest:
        assert not out.t[2].any()
    else:
        assert bool((out.t[2] == 9.0).all())


@gpu
@pytest.mark.parametrize("rows", [[2, 1], [17, 9], [60, 45], [1, 0]])
@pytest.mark.parametrize("pages", [1, 8, 40])
@pytest.mark.parametrize("tail", [1, 130])
def test_rows_behind_the_last_sequence_of_a_prefix_alone(rows, pages, tail):
    """All pages shared, so that no sequence has keys of its own: tables of one split and
    of several, 16-row and 128-row tiles, padding that fills tiles of its own."""
    p = Paged(rows, [0, 0], heads=12, tail=tail)
    p.k_pages, p.v_pages = (p.randn(pages, 2, 16, 64) for _ in range(2))
    p.table = torch.arange(pages, dtype=torch.int32, device=p.q.device).expand(2, pages)
    p.used, p.shared = [list(range(pages))] * 2, pages
    p.lengths_list = [max(16 * pages - 5, rows[0]), max(16 * pages - 11, rows[1])]
    if pages == 1:  # (no row past the table; those before the sequence's start give zeros)
        p.lengths_list = [min(n, 16) for n in p.lengths_list]
    p.lengths.copy_(torch.tensor(p.lengths_list))
    want, slack = p.reference()
    got = p.attention()
    _near(got[:p.total], want[:p.total], slack[:p.total])
    assert not got[p.total:].any()
    out = Guarded(*p.q.shape, value=7.0)
    p.attention(out=out.t)
    assert torch.equal(out.t[:p.total], got[:p.total])
    assert bool((out.t[p.total:] == 7.0).all()) and out.kept()
    p.cu.zero_()  # no rows at all
    out.t.fill_(7.0)
    p.attention(out=out.t)
    assert bool((out.t == 7.0).all()) and not p.attention().any()


# ---- verification over rows of few entries ----

@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [4097, 33000, 151936])
def test_verify_on_a_border_before_spans_without_weight(vocab, dtype):
    """Two entries of 2^-54 before two halves, 1024 apart, and a share of one half: the
    first half's running sum, 2^-53 above it, passes.  (The lanes' sums in other orders
    are 0.5 and, over the empty span behind it, 0.5 + 2^-53.)  Then entries of one lane's
    several spans, and each entry alone."""
    target = torch.zeros(1, 1, vocab, dtype=dtype, device="cuda")
    target[0, 0, [0, 1024]] = 2.0 ** -54
    target[0, 0, [2048, 4096]] = 0.5
    none = torch.zeros(1, 0, dtype=torch.int64, device="cuda")
    for u in (0.5, 0.5 - 2.0 ** -24, 0.5 + 2.0 ** -24, 0.0, 2.0 ** -60, 1.0):
        share = torch.full((1, 1), u, device="cuda")
        _same(verify_drafts_hip(target, none, share), _verified(target, none, share, None))
    for at in [*range(0, vocab, 1021), vocab - 1]:
        target.zero_()
        target[0, 0, at] = 2.0 ** -20
        for u in (0.0, 1.0 - 2.0 ** -24):
            got = verify_drafts_hip(target, none, torch.full((1, 1), u, device="cuda"))
            assert got[0].tolist() == [[at]], (at, u)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("batch, vocab", [(5, 5000), (3, 40000), (2, 151936), (260, 32000)])
@pytest.mark.parametrize("kept", [1, 2, 20])
def test_verify_of_rows_cut_to_their_largest(dtype, batch, vocab, kept):
    """Probabilities cut to the largest few of a row, most spans empty, with a draft cut
    to others; uniforms at zero, next to one, and between."""
    gen = torch.Generator(device="cuda").manual_seed(vocab + kept)

    def cut(rows):
        x = torch.rand(batch, rows, kept, generator=gen, device="cuda") + 0.05
        at = torch.rand(batch, rows, vocab, generator=gen, device="cuda").topk(kept, -1).indices
        return torch.zeros(batch, rows, vocab, device="cuda").scatter_(-1, at, x / x.sum(-1, True)).to(dtype), at

    target, at = cut(3)
    draft, drafted = cut(2)
    tokens = torch.where(torch.rand(batch, 2, generator=gen, device="cuda") < 0.5, at[:, :2, 0], drafted[:, :, 0])
    uniforms = torch.rand(batch, 3, generator=gen, device="cuda")
    uniforms[::3, 2], uniforms[1::3, 2] = 0.0, 1.0 - 2.0 ** -24
    for q in (draft, None):
        got = verify_drafts_hip(target, tokens, uniforms, draft_probs=q)
        _same(got, _verified(target, tokens, uniforms, q))
        chosen = got[0].gather(1, got[1].long().view(-1, 1))
        weight = target[torch.arange(batch, device=target.device), got[1].long()].gather(1, chosen)
        assert bool((chosen >= 0).all() and (weight > 0).all())


# ---- values that are not finite, at keys of hardly any weight ----

@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("rows, past, shared, spots", [
    ([1], [100], 0, [40]), ([2], [900], 0, [0, 500]), ([1, 1], [300, 40], 9, [3, 150]), ([60, 1], [2000, 7], 0, [64, 1033]),
    ([40], [100], 40, [100, 600])])
def test_values_that_are_not_finite_at_keys_of_little_weight(dtype, bad, rows, past, shared, spots):
    """Scores of the 64 keys around a spot some 10^-125 below the others: whichever wave
    or split has them alone, an infinity or NaN among their values reaches the rows that
    see it (the formula's weight is not zero), and its dimension only."""
    p = Paged(rows, past, heads=12, dim=64, shared=shared, dtype=dtype)
    p.q.copy_(1.0 + p.randn(*p.q.shape) / 16)
    for b, length in enumerate(p.lengths_list):
        where = torch.tensor(p.used[b], device=p.q.device)[:-(-length // 16)]
        p.k_pages[where] = 4.0 + p.randn(len(where), 2, 16, 64) / 16
    for spot in spots:
        first = max(0, spot // 32 * 32 - 32)
        for t in range(first, min(first + 96, p.lengths_list[0] - rows[0])):
            p.k_pages[p.used[0][t // 16], :, t % 16] = -32.0
    want, slack = p.reference()  # (finite: a library product with an infinity may give NaN)
    for spot in spots:
        p.v_pages[p.used[0][spot // 16], :, spot % 16, 9] = bad
    want[:None if spots[0] < 16 * shared else rows[0], :, 9] = bad
    _near(p.attention(), want, slack)


# ---- values of any size ----

@gpu
@pytest.mark.parametrize("rows, past, batch, shared", [
    ([1], [1023], 400, 0), ([2], [1022], 1, 0), ([260], [900], 1, 0), ([70], [30], 2, 64)])
@pytest.mark.parametrize("size", [2.0 ** 117, 2.0 ** -110])
def test_values_of_any_size(rows, past, batch, shared, size):
    """Scores that rise by nearly eight units of the base-2 exponent after every wave's
    first keys, and values whose sum over the keys fp32 just holds (2^117 times a
    thousand to two thousand), then small ones.  Many sequences over the same pages:
    one split."""
    p = Paged(rows, past, heads=12, dim=64, shared=shared)
    p.q.fill_(1.0)
    length = p.lengths_list[0]
    where = torch.tensor(p.used[0], device=p.q.device)
    p.k_pages[where] = 0.6  # (0.6 * 64 / 8 = 4.8: 6.9 units of the base-2 exponent)
    for first in range(0, length, 1024):
        p.k_pages[where[first // 16:(first + 128) // 16]] = 0.0
    p.v_pages[where] = ((1.0 + torch.rand(len(where), 2, 16, 64, device=p.q.device) / 2) * size).to(BF16)
    want, slack = p.reference()
    assert bool(want.isfinite().all())
    if batch > 1:
        p.q = p.q.repeat(batch, 1, 1)
        p.table = p.table.expand(batch, -1)
        p.cu = torch.arange(batch + 1, dtype=torch.int32, device=p.q.device) * rows[0]
        p.lengths = p.lengths.repeat(batch)
        want, slack = want.repeat(batch, 1, 1), slack.repeat(batch, 1, 1)
    _near(p.attention(), want, slack)


# ---- outputs beside their inputs ----

@gpu
def test_append_into_outputs_beside_its_inputs():
    """What lies apart is taken, wherever it lies: an output of its own for queries and
    keys of one tensor, heads of q, k and v in turn, an output between the queries' heads,
    keys and values in turn behind the queries."""
    p = Paged([3, 2], [7, 0], heads=2)
    inv = torch.rand(32, device="cuda")

    def append(q, k, v, out=None):
        return paged_append_hip(q, k, v, p.k_pages, p.v_pages, p.table, p.cu, p.lengths, inv, out=out)

    def caches():
        return [c.view(torch.int16).clone() for c in (p.k_pages, p.v_pages)]

    def same(got, q, k, v):
        """The call's outputs against those for copies of its inputs."""
        left = caches()
        assert torch.equal(got, append(q.clone(), k.clone(), v.clone()))
        assert all(torch.equal(a, b) for a, b in zip(left, caches()))

    one = p.randn(5, 2, 64)
    kept = one.clone()
    same(append(one, one, one, torch.empty_like(one)), one, one, one)
    assert torch.equal(one, kept)
    for fused in (p.randn(5, 2, 3, 64), p.randn(5, 3, 2, 64).transpose(1, 2)):
        q, k, v = (fused[:, :, i] for i in range(3))
        before = q.clone()
        got = append(q, k, v, q)
        assert got.data_ptr() == q.data_ptr()
        same(got, before, k, v)
        before, other = k.clone(), v.clone()
        same(append(q, k, k, v), q, k, k)  # (over v's place)
        assert torch.equal(k, before) and not torch.equal(v, other)
    rows = p.randn(5, 6, 64)
    q, k, v = rows[:, :2], rows[:, 2::2], rows[:, 3::2]
    before = q.clone()
    same(append(q, k, v, q), before, k, v)
    rows = p.randn(5, 6, 64)
    for out in (rows[:, 1:3], rows[:, 1:5:2], rows[:, 3:5]):
        with pytest.raises(ValueError, match="out must be q itself"):
            append(rows[:, :2], rows[:, 2:4], rows[:, 4:], out)
    with pytest.raises(ValueError, match="must not share its rows"):
        append(rows[:, :2], rows[:, 1:3], rows[:, 4:], rows[:, :2])


@gpu
def test_attention_into_an_output_between_the_queries():
    p = Paged([3, 1], [20, 5], heads=4, shared=1)
    want = p.attention()
    both = torch.zeros(4, 4, 2, 64, dtype=BF16, device="cuda")
    both[:, :, 0] = p.q
    p.attention(q=both[:, :, 0], out=both[:, :, 1])
    assert torch.equal(both[:, :, 1], want) and torch.equal(both[:, :, 0], p.q)
    with pytest.raises(ValueError, match="share no memory"):
        p.attention(q=both[:, :, 0], out=both.view(4, 8, 64)[:, 2:6])


# ---- limits of shapes ----

@gpu
def test_limits_of_shapes_are_value_errors():
    def z(*shape, dtype=BF16):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    cu, lengths = torch.tensor([0, 2], dtype=torch.int32, device="cuda"), z(1, dtype=torch.int32)
    for dim in (32, 72, 80, 256):
        with pytest.raises(ValueError, match="head_dim of 64 or 128"):
            paged_attention_hip(z(2, 4, dim), z(3, 2, 16, dim), z(3, 2, 16, dim), z(1, 3, dtype=torch.int32), cu, lengths)
    for dim in (72, 272):
        with pytest.raises(ValueError, match="head_dim that is a multiple of 16 up to 256"):
            paged_append_hip(z(2, 4, dim), z(2, 2, dim), z(2, 2, dim), z(3, 2, 16, dim), z(3, 2, 16, dim),
                             z(1, 3, dtype=torch.int32), cu, lengths, None)
    pool = [z(1, 1, 1 << 20, 64) for _ in range(2)]
    with pytest.raises(ValueError, match="at most 2.31 - 2.20 positions"):
        paged_attention_hip(z(2, 1, 64), *pool, z(1, 2048, dtype=torch.int32), cu, lengths)
    with pytest.raises(ValueError, match="page_size must be a power of two"):
        paged_attention_hip(z(2, 1, 64), z(1, 1, 24, 64), z(1, 1, 24, 64), z(1, 2, dtype=torch.int32), cu, lengths)
    with pytest.raises(ValueError, match="shared_pages must be in"):
        paged_attention_hip(z(2, 1, 64), *pool, z(1, 2, dtype=torch.int32), cu, lengths, shared_pages=3)
    far = torch.empty(15 * (1 << 25) + 64, dtype=BF16, device="cuda").as_strided((1, 1, 16, 64), (0, 0, 1 << 25, 1))
    with pytest.raises(ValueError, match="position strides must be at most 2.24"):
        paged_attention_hip(z(2, 1, 64), far, z(1, 1, 16, 64), z(1, 2, dtype=torch.int32), cu, lengths)


# ---- row bounds that fall or lead out, with everything around the buffers watched ----

@gpu
@pytest.mark.parametrize("values", [[-7, 90, 2, -1], [5, 5, 5, 5], [0, 2 ** 31 - 1, -(2 ** 31), 4], [0, 2, 3, 2 ** 31 - 1],
                                    [0, 0, 0, -(2 ** 31)], [2 ** 31 - 1] * 4, [0, 4, 0, 4], [3, 2, 1, 0]])
@pytest.mark.parametrize("rows, shared", [([2, 1, 1], 2), ([2, 1, 1], 0), ([60, 1, 50], 0), ([60, 1, 50], 9)])
def test_row_bounds_that_fall_or_lead_out_write_nothing_else(values, rows, shared):
    """Whatever cu_rows holds: rows behind its last entry keep what they hold, and nothing
    around the output, the pools and the rotated queries is written, nor a page that no
    table entry names."""
    p = Paged(rows, [3, 40, 9], shared=shared, heads=12)
    scale = p.total // 4  # (bounds inside the rows at both sizes)
    p.cu.copy_(torch.tensor([v * scale if 0 < v < 100 else v for v in values], dtype=torch.int64).to(torch.int32))
    pools = [Guarded(*c.shape, value=5.0) for c in (p.k_pages, p.v_pages)]
    for pool, cache in zip(pools, (p.k_pages, p.v_pages)):
        pool.t.copy_(cache.nan_to_num(0.25))
    before = [pool.t.clone() for pool in pools]
    end = max(int(p.cu[-1]), 0)
    k, v = p.randn(p.total, 2, 64), p.randn(p.total, 2, 64)
    turned = Guarded(*p.q.shape, value=7.0)
    paged_append_hip(p.q, k, v, pools[0].t, pools[1].t, p.table, p.cu, p.lengths, None, out=turned.t)
    assert turned.kept() and bool((turned.t[end:] == 7.0).all())
    named = torch.zeros(p.k_pages.shape[0], dtype=torch.bool, device="cuda")
    named[[page for used in p.used for page in used]] = True
    for pool, old in zip(pools, before):
        assert pool.kept() and torch.equal(pool.t[~named], old[~named])
    after = [pool.t.clone() for pool in pools]
    out = Guarded(*p.q.shape, value=7.0)
    paged_attention_hip(p.q, pools[0].t, pools[1].t, p.table, p.cu, p.lengths, shared_pages=shared, out=out.t)
    assert out.kept() and bool((out.t[end:] == 7.0).all())
    fresh = paged_attention_hip(p.q, pools[0].t, pools[1].t, p.table, p.cu, p.lengths, shared_pages=shared)
    assert not fresh[end:].any()
    for pool, old in zip(pools, after):
        assert pool.kept() and torch.equal(pool.t, old)


# ---- tables wider than the sequences, long sequences ----

@gpu
@pytest.mark.parametrize("columns", [1, 60, 2000])
@pytest.mark.parametrize("rows, past, more", [
    ([1, 1, 1], [3, 200, 31], {"dim": 128, "heads": 12}),
    ([1] * 5, [0, 2, 15, 16, 300], {"shared": 9, "heads": 8, "dtype": F16}),
    ([70, 1, 33], [0, 400, 5], {"heads": 12, "dim": 128, "page": 32}),
    ([60, 30], [64, 7], {"shared": 21, "heads": 12, "dim": 64}),
])
def test_tables_wider_than_their_sequences(rows, past, more, columns):
    """Columns behind the longest sequence, as a captured graph's table has them: what they
    hold (no page, or any) is not looked at."""
    p = Paged(rows, past, **more)
    want, slack = p.reference()
    spare = torch.full((len(rows), columns), -1, dtype=torch.int32, device="cuda")
    spare[:, ::3] = 2 ** 31 - 1
    spare[:, 1::3] = 0
    p.table = torch.cat((p.table, spare), 1)
    _near(p.attention(), want, slack)


@gpu
@pytest.mark.parametrize("rows, past, heads, dim, dtype", [(1, 20000, 12, 128, BF16), (3, 33333, 8, 64, F16),
                                                           (30, 9000, 12, 64, BF16)])
def test_attention_over_one_long_sequence(rows, past, heads, dim, dtype):
    p = Paged([rows], [past], heads=heads, dim=dim, page=128, dtype=dtype)
    _near(p.attention(), *p.reference())
