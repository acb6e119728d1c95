"""The packed prompt attention (qwen_int4_hip.packed) and the page operators
(qwen_int4_hip.pages) against plain implementations, and what they refuse.

Tolerances count roundings: a result in 16 bits is off by at most finfo.eps / 2 of its
value, a probability likewise, and what fp32 adds is bounded beside the comparison."""

from __future__ import annotations

import ctypes
import math
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))

from test_packed_lanes import POOLS, compacted, forked, resized, state_of  # noqa: E402

import qwen_int4_hip  # noqa: E402
from qwen_int4_hip import (  # noqa: E402
    _lib, packed_attention_hip, paged_append_hip, paged_attention_hip, paged_compact_hip, paged_fork_hip, paged_resize_hip)

BF16, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32

built = pytest.mark.skipif(not _lib.library_built(), reason="HIP library not built (run __graft_entry__.build())")


def gpu(test):
    return pytest.mark.gpu(pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a ROCm GPU")(built(test)))


def ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int64).to(I32).to(device)


# ---------------------------------------------------------------------------
# On the CPU: the refusals
# ---------------------------------------------------------------------------

def _prompt(dtype=BF16, rows=5, heads=4, kv_heads=2, dim=64, batch=2):
    return {"q": torch.zeros(rows, heads, dim, dtype=dtype), "k": torch.zeros(rows, kv_heads, dim, dtype=dtype),
            "v": torch.zeros(rows, kv_heads, dim, dtype=dtype), "cu_rows": torch.zeros(batch + 1, dtype=I32)}


@built
def test_attention_refuses_before_launch():
    good = _prompt()
    for change, error, said in [
            ({"q": torch.zeros(5, 4, 64)}, TypeError, "q must have dtype"),
            ({"k": torch.zeros(5, 2, 64, dtype=F16)}, TypeError, "k must have the dtype of q"),
            ({"v": torch.zeros(5, 2, 64, dtype=F16)}, TypeError, "v must have the dtype of q"),
            ({"k": torch.zeros(4, 2, 64, dtype=BF16)}, ValueError, "k must have shape"),
            ({"v": torch.zeros(5, 1, 64, dtype=BF16)}, ValueError, "v must have shape"),
            ({"v": torch.zeros(5, 2, 128, dtype=BF16)}, ValueError, "v must have shape"),
            ({"q": torch.zeros(5, 256, dtype=BF16)}, ValueError, "q must have 3 dimensions"),
            ({"cu_rows": torch.zeros(3, dtype=torch.int64)}, TypeError, "cu_rows must have dtype"),
            ({"cu_rows": torch.zeros(0, dtype=I32)}, ValueError, "at least one entry"),
            ({"scale": "1"}, TypeError, "scale must be a number"),
            ({"scale": torch.tensor(1.0)}, TypeError, "scale must be a number"),
            ({"out": torch.zeros(5, 4, 64)}, TypeError, "out must have q's dtype"),
            ({"out": torch.zeros(5, 2, 64, dtype=BF16)}, ValueError, "out must have q's shape"),
            ({"out": torch.zeros(5, 64, 4, dtype=BF16).transpose(1, 2)}, ValueError, "out must be 16-byte aligned"),
            ({"out": torch.zeros(1, 4, 64, dtype=BF16).expand(5, 4, 64)}, ValueError, "out must be 16-byte aligned"),
            ({"q": torch.zeros(5, 4, 64, dtype=BF16).requires_grad_()}, RuntimeError, "has no gradient"),
            ({"q": [1.0]}, TypeError, "q must be a torch.Tensor"),
            ({}, ValueError, "q must be a GPU tensor")]:
        with pytest.raises(error, match=said):
            packed_attention_hip(**(good | change))


@built
def test_page_operators_refuse_before_launch():
    table, lengths, users = torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32), torch.zeros(6, dtype=I32)
    resize = {"page_table": table, "lengths": lengths, "page_users": users, "page_size": 16}
    pool = torch.zeros(6, 2, 16, 64, dtype=BF16)
    compact = {"k_pages": pool, "v_pages": pool.clone(), "page_table": table, "page_users": users}
    fork = compact | {"lengths": lengths, "parents": torch.zeros(4, dtype=I32)}
    indices = [
        ({"page_table": table.long()}, TypeError, "page_table must have dtype torch.int32"),
        ({"page_table": table[0]}, ValueError, "page_table must have 2 dimensions"),
        ({"page_table": table[:, :0]}, ValueError, "at least one column"),
        ({"page_users": users.long()}, TypeError, "page_users must have dtype torch.int32"),
        ({}, ValueError, "must be a GPU tensor"),
    ]
    rows = [
        ({"lengths": lengths.long()}, TypeError, "lengths must have dtype torch.int32"),
        ({"lengths": torch.zeros(3, dtype=I32)}, ValueError, r"lengths must have shape \[2\]"),
    ]
    deep = torch.zeros(3, 6, 2, 16, 64, dtype=BF16)
    pools = [
        ({"k_pages": pool.float()}, TypeError, "k_pages must have dtype"),
        ({"v_pages": pool.half()}, TypeError, "v_pages must have the dtype"),
        ({"v_pages": torch.zeros(6, 2, 32, 64, dtype=BF16)}, ValueError, "v_pages must have the shape"),
        ({"k_pages": pool[0]}, ValueError, "k_pages must have 4 dimensions"),
        ({"k_pages": deep}, ValueError, "v_pages must have the shape"),
        ({"v_pages": pool}, ValueError, "must not share memory"),
        ({"k_pages": deep[:2], "v_pages": deep[1:]}, ValueError, "must not share memory"),
        ({"k_pages": deep[0], "v_pages": deep[1]}, ValueError, "must be a GPU tensor"),
        ({"k_pages": pool[:1].expand(6, 2, 16, 64)}, ValueError, "no two entries in one place"),
        ({"k_pages": torch.zeros(6, 2, 16, 68, dtype=BF16)[..., :64]}, ValueError, "k_pages must be 16-byte"),
        ({"page_users": torch.zeros(5, dtype=I32)}, ValueError, r"page_users must have shape \[6\]"),
        ({"k_pages": pool.requires_grad_(False).clone().requires_grad_()}, RuntimeError, "has no gradient"),
    ]
    for call, good, changes in [
            (paged_resize_hip, resize, indices + rows + [
                ({"page_size": 16.0}, TypeError, "page_size must be an integer"),
                ({"page_size": True}, TypeError, "page_size must be an integer"),
                ({"page_size": 2 ** 70}, ValueError, "out of range"),
                ({"page_users": users[:0]}, ValueError, "at least one entry")]),
            (paged_fork_hip, fork, indices + rows + pools + [
                ({"parents": torch.zeros(4, dtype=torch.int64)}, TypeError, "parents must have dtype"),
                ({"parents": torch.zeros(2, 2, dtype=I32)}, ValueError, "parents must have 1 dimensions")]),
            (paged_compact_hip, compact, indices + pools)]:
        for change, error, said in changes:
            with pytest.raises(error, match=said):
                call(**(good | change))


@built
def test_c_entry_points_refuse_before_launch():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buffer) + 15) & ~15
    null, f = None, ctypes.c_float
    row = ctypes.byref(_lib.Rows(p, 128, 64))

    def attention(q=row, k=row, v=row, out=row, cu=p, batch=1, rows=1, heads=4, kv_heads=2, dim=64, dtype=2, scale=0.1):
        return lib.qwen2_packed_attention(q, k, v, out, cu, batch, rows, heads, kv_heads, dim, dtype, f(scale), 1, null)

    assert attention(dtype=3) == _lib.STATUS_INVALID_DTYPE and attention(dim=96) == _lib.STATUS_UNSUPPORTED
    assert attention(heads=3) == 1 and attention(heads=0) == 1 and attention(kv_heads=0) == 1 and attention(rows=-1) == 1
    assert attention(batch=-1) == 1 and attention(scale=math.inf) == 1 and attention(scale=math.nan) == 1
    assert attention(cu=null) == 1 and attention(cu=p + 2) == 1
    for bad in (null, ctypes.byref(_lib.Rows(null, 128, 64)), ctypes.byref(_lib.Rows(p + 2, 128, 64)),
                ctypes.byref(_lib.Rows(p, 128, 60))):
        assert attention(q=bad) == 1 and attention(k=bad) == 1 and attention(v=bad) == 1 and attention(out=bad) == 1
    assert attention(k=ctypes.byref(_lib.Rows(p, 1 << 25, 64))) == _lib.STATUS_UNSUPPORTED
    assert attention(v=ctypes.byref(_lib.Rows(p, -128, 64))) == _lib.STATUS_UNSUPPORTED
    assert attention(rows=1 << 26, heads=32) == _lib.STATUS_UNSUPPORTED
    assert attention(rows=0) == _lib.STATUS_OK and attention(batch=0) == _lib.STATUS_OK

    def resize(table=p, users=p, batch=2, width=3, pages=6, page=16, ws=p, nbytes=1 << 12):
        return lib.qwen2_paged_resize(table, 3, p, users, p, p, p, batch, width, pages, page, ws, nbytes, null)

    assert resize(batch=-1) == 1 and resize(width=0) == 1 and resize(pages=0) == 1 and resize(batch=(1 << 20) + 1) == 1
    assert resize(page=8) == 1 and resize(page=48) == 1 and resize(page=1 << 21) == 1
    assert resize(pages=(1 << 24) + 1) == _lib.STATUS_UNSUPPORTED
    assert resize(batch=1 << 20, width=1 << 12) == _lib.STATUS_UNSUPPORTED
    assert resize(table=null) == 1 and resize(users=p + 2) == 1
    need = lib.qwen2_paged_resize_workspace_bytes(2, 3, 20000)
    assert need > 0 and resize(pages=20000, nbytes=need - 1) == _lib.STATUS_WORKSPACE
    assert resize(pages=20000, ws=null) == _lib.STATUS_WORKSPACE
    assert lib.qwen2_paged_resize_workspace_bytes(2, 0, 6) == 0 and lib.qwen2_paged_resize_workspace_bytes(2, 3, 6) == 0

    def pool(**change):
        fields = {"k": p, "v": p, "k_layer": 0, "k_page": 2048, "k_head": 1024, "k_position": 64, "v_layer": 0, "v_page": 2048,
                  "v_head": 1024, "v_position": 64, "layers": 1, "num_pages": 6, "kv_heads": 2, "page_size": 16, "head_dim": 64}
        return ctypes.byref(_lib.PagePool(**(fields | change)))

    def fork(c, batch=2, children=4, width=3, parents=p, ws=p, nbytes=1 << 12):
        return lib.qwen2_paged_fork(c, p, 3, p, p, parents, p, p, p, p, batch, children, width, ws, nbytes, null)

    def compact(c, batch=2, width=3, users=p, ws=p, nbytes=1 << 12):
        return lib.qwen2_paged_compact(c, p, 3, users, p, p, p, batch, width, ws, nbytes, null)

    for call in (fork, compact):
        for change, status in [({"k": null}, 1), ({"v": p + 8}, 1), ({"layers": 0}, 1), ({"kv_heads": 0}, 1), ({"page_size": 24}, 1),
                               ({"k_head": 60}, 1), ({"v_page": -8}, 1), ({"num_pages": 0}, 1),
                               ({"num_pages": (1 << 24) + 1}, _lib.STATUS_UNSUPPORTED),
                               ({"head_dim": 60}, _lib.STATUS_UNSUPPORTED), ({"head_dim": 2048}, _lib.STATUS_UNSUPPORTED)]:
            assert call(pool(**change)) == status, (call, change, lib.w4g64_last_error())
        assert call(null) == 1 and call(pool(), batch=-1) == 1 and call(pool(), width=0) == 1
        assert call(pool(num_pages=20000), ws=null) == call(pool(num_pages=20000), nbytes=8) == _lib.STATUS_WORKSPACE
    assert fork(pool(), children=-1) == 1 and fork(pool(), parents=null) == 1
    assert compact(pool(), users=null) == 1


# ---------------------------------------------------------------------------
# Attention on the GPU
# ---------------------------------------------------------------------------

class Prompts:
    """Packed rows, parts of one fused projection; `tail` rows of no sequence behind them."""

    def __init__(self, lengths, *, heads=4, kv_heads=2, dim=64, dtype=BF16, tail=0, seed=0):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lengths, self.total, self.dtype = lengths, sum(lengths), dtype
        qkv = torch.randn(self.total + tail, heads + 2 * kv_heads, dim, generator=self.gen, device="cuda").to(dtype)
        self.q, self.k, self.v = qkv.split((heads, kv_heads, kv_heads), 1)
        self.cu = ints([sum(lengths[:b]) for b in range(len(lengths) + 1)])

    def attention(self, **more):
        return packed_attention_hip(self.q, self.k, self.v, self.cu, **more)

    def reference(self, scale=None):
        """(attended rows, bound of what is off before the result's rounding), 64 bits."""
        q, k, v = (t.double() for t in (self.q, self.k, self.v))
        group, dim, at = q.shape[1] // k.shape[1], q.shape[2], 0
        scale = dim ** -0.5 if scale is None else scale
        out, slack = torch.zeros_like(q), torch.zeros_like(q)
        half = torch.finfo(self.dtype).eps / 2
        for n in self.lengths:
            if n:
                x = q[at:at + n].transpose(0, 1)
                y, z = (t[at:at + n].transpose(0, 1).repeat_interleave(group, 0) for t in (k, v))
                hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
                w = torch.softmax((x @ y.transpose(1, 2) * scale).masked_fill(hidden, -math.inf), dim=-1)
                part, size = w @ z, w @ z.abs()
                # a score: dim products and additions, the scale's and the exponential's roundings; a
                # probability: half a step, in the sum and in the sum that divides it, so that what a value
                # differs from the mean by counts (size + |part| at most); sums over the keys in blocks of 8;
                # probabilities of fp16 under 2^-25 of the largest are off by 2^-36 of it
                big = (x.abs() @ y.abs().transpose(1, 2)).amax() * abs(scale)
                rel = 2.0 ** -24 * (2 * (dim + 8) * big + n / 4 + 64)
                rare = n * 2.0 ** -36 * z.abs().amax()
                out[at:at + n] = part.transpose(0, 1)
                slack[at:at + n] = (rel * size + half * (1 + 2 * half) * (size + part.abs()) + rare).transpose(0, 1)
            at += n
        return out, slack


def near(got, want, slack):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half  # (a subnormal result's half step)
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    off = torch.where(want.isnan() | (got == want), 0.0, (got - want).abs() - (want.abs() * half + slack * (1 + half) + tiny))
    assert float(off.nan_to_num(nan=1e9).amax() if off.numel() else 0) <= 0, float(off.amax())


PROMPTS = [
    ([1], {}),
    ([2, 1], {"dim": 128, "dtype": F16}),
    ([37], {"heads": 12, "dim": 128}),
    ([31, 32, 33], {"heads": 2}),
    ([63, 64, 65], {"heads": 2, "kv_heads": 1, "dim": 128}),
    ([5, 0, 0, 17, 0], {"heads": 14, "kv_heads": 2}),
    ([127, 128, 129], {"heads": 3, "kv_heads": 3, "dtype": F16}),
    ([512], {"heads": 12, "dim": 128}),
    ([700], {"heads": 9, "kv_heads": 3, "dim": 64, "dtype": F16}),
    ([1100], {"heads": 12, "dim": 128}),
    ([1500], {"heads": 16, "kv_heads": 16, "dim": 64}),
    ([2049], {"heads": 12, "dim": 128, "dtype": F16}),
    ([300, 1, 700, 64, 255], {"heads": 32, "kv_heads": 8, "dim": 128}),
    ([1000, 3, 411], {"heads": 8, "kv_heads": 1, "dim": 64}),
    ([b % 97 for b in range(80)], {"heads": 16, "kv_heads": 16, "dim": 64, "dtype": F16}),
    ([(37 * b) % 150 for b in range(64)], {"heads": 12, "dim": 128}),
    ([1] * 200, {"heads": 6, "kv_heads": 2, "dim": 128}),
    ([b % 4 for b in range(700)], {"heads": 2, "dim": 64}),
    ([0] * 300 + [5, 130] + [0] * 250 + [1], {"heads": 8, "kv_heads": 2, "dim": 128, "dtype": F16}),
    ([3, 150], {"heads": 64, "kv_heads": 1, "dim": 64}),
    ([90, 1], {"heads": 1, "kv_heads": 1, "dim": 128}),
    ([1900, 600], {"heads": 40, "kv_heads": 8, "dim": 128, "dtype": F16}),
    ([30 + 3 * b for b in range(66)], {"heads": 12, "dim": 128}),
    ([260] * 40, {"heads": 12, "dim": 64}),
    ([1200] + [20] * 30, {"heads": 8, "kv_heads": 1, "dim": 128}),
]


@gpu
@pytest.mark.parametrize("lengths, more", PROMPTS)
def test_attention_is_the_formula(lengths, more):
    p = Prompts(lengths, **more)
    near(p.attention(), *p.reference())


@gpu
def test_attention_is_the_same_for_every_form():
    """One sequence in calls whose other sequences and heads choose other workgroups."""
    for dtype, dim in ((BF16, 128), (F16, 64)):
        p = Prompts([257], heads=2, kv_heads=2, dim=dim, dtype=dtype)
        want, slack = p.reference()
        near(p.attention(), want, slack)
        for copies, times in ((1, 20), (4, 4), (40, 2), (3, 60)):
            q, k, v = (t.repeat(copies, times, 1) for t in (p.q, p.k, p.v))
            got = packed_attention_hip(q, k, v, ints([257 * c for c in range(copies + 1)]))
            near(got, want.repeat(copies, times, 1), slack.repeat(copies, times, 1))


@gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_scales(scale, dtype):
    p = Prompts([40, 1, 133], dtype=dtype, dim=128)
    near(p.attention(scale=scale), *p.reference(scale=scale))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_over_far_apart_scores(dtype):
    """Most keys far below the maximum; then one key that outweighs all others."""
    p = Prompts([900], dtype=dtype)
    p.q[:, :] = torch.where(torch.rand(p.q.shape, generator=p.gen, device="cuda") < 0.7, 0.1, 0.9).to(dtype)
    near(p.attention(), *p.reference())
    for spot in (0, 450, 899):
        kept = p.k[spot].clone()
        p.k[spot] = 12.0
        near(p.attention(), *p.reference())
        p.k[spot] = kept


@gpu
@pytest.mark.parametrize("lengths", [[2, 0, 1], [70, 200], [600]])
def test_rows_behind_the_last_sequence(lengths):
    p = Prompts(lengths, tail=3, heads=6)
    want, slack = p.reference()
    got = p.attention()
    near(got, want, slack)
    assert not got[p.total:].any()
    out = torch.full_like(got, 7.0)
    assert p.attention(out=out) is out
    assert torch.equal(out[:p.total], got[:p.total]) and bool((out[p.total:] == 7.0).all())


@gpu
@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("lengths, heads", [([20, 30], 4), ([5, 400, 70], 4), ([300], 40), ([130] * 30, 12), ([290] * 30, 12)])
def test_values_that_are_not_finite(dtype, dim, bad, lengths, heads):
    """Whole values at one position: the rows before it and the other sequences are
    unmoved, those from it on are what the formula says; then one element alone, then two
    that have no sum; then a key."""
    p = Prompts(lengths, heads=heads, kv_heads=2, dim=dim, dtype=dtype)
    want, slack = p.reference()
    which = min(1, len(lengths) - 1)
    begin, end = sum(lengths[:which]), sum(lengths[:which + 1])
    spot = begin + lengths[which] * 3 // 5
    seen = torch.zeros(p.total, dtype=torch.bool, device="cuda")
    seen[spot:end] = True

    def check(touched, value):
        got = p.attention()
        assert bool((got[touched].isnan() if math.isnan(value) else got[touched] == value).all())
        near(torch.where(touched, 0, got), torch.where(touched, 0.0, want), slack)

    kept = p.v[spot].clone()
    p.v[spot] = bad
    check(seen.view(-1, 1, 1).expand(p.q.shape).clone(), bad)
    p.v[spot] = kept
    touched = torch.zeros(p.q.shape, dtype=torch.bool, device="cuda")
    touched[spot:end, heads // 2:, 7] = True
    p.v[spot, 1, 7] = bad
    check(touched, bad)
    p.v[begin, 1, 7] = -bad
    first = touched.clone()
    first[begin:spot, heads // 2:, 7] = True
    got = p.attention()
    assert bool(got[touched].isnan().all()) and not got[first].isfinite().any()
    near(torch.where(first, 0, got), torch.where(first, 0.0, want), slack)
    p.v[spot], p.v[begin, 1, 7] = kept, 0.25
    want, slack = p.reference()
    p.k[spot] = bad  # (of its own sequence's rows only those from it on can see it)
    got = p.attention()
    near(got[~seen], want[~seen], slack[~seen])
    if math.isnan(bad):
        assert bool(got[seen].isnan().all())


@gpu
def test_an_infinity_of_hardly_any_weight_reaches_its_rows():
    """Its key is so far below the others that its weight is zero in fp32; its keys' block is
    another wave's, another tile's, or the same."""
    for spot in (0, 40, 70, 130):
        p = Prompts([200], heads=2, kv_heads=1, dim=64)
        p.q[:], p.k[:] = 4.0, 4.0
        p.k[spot] = -4.0
        p.v[spot, 0, 3] = math.inf
        got = p.attention()
        assert bool((got[spot:, :, 3] == math.inf).all()) and bool(got[:spot].isfinite().all())
        got[spot:, :, 3] = 0
        assert bool(got.isfinite().all())


@gpu
def test_large_values_add_up_as_far_as_fp32_goes():
    p = Prompts([300], heads=2, kv_heads=1, dim=64)
    p.v[:] = 1e36
    near(p.attention(), *p.reference())


@gpu
@pytest.mark.parametrize("values", [[-7, 90, 2, -1], [5, 5, 5, 5], [0, 2 ** 31 - 1, -(2 ** 31), 4], [2 ** 31 - 1] * 4])
def test_row_bounds_that_fall_or_lead_out_stay_in_the_buffers(values):
    p = Prompts([2, 1, 1], heads=6)
    p.cu.copy_(ints(values))
    out = torch.full_like(p.q, 7.0)
    p.attention(out=out)
    p.attention()
    end = min(max(values[-1], 0), 4)
    assert bool((out[end:] == 7.0).all())


@gpu
def test_attention_reads_strided_and_unaligned_rows():
    p = Prompts([70, 9], heads=4, dim=64)
    want = p.attention()
    rows = p.total
    odd = [torch.zeros(t.numel() + 3, dtype=BF16, device="cuda")[3:].view(t.shape).copy_(t) for t in (p.q, p.k, p.v)]
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (p.q, p.k, p.v)]
    apart = [torch.zeros(rows, 9, 2 * 64, dtype=BF16, device="cuda")[:, 1:1 + 2 * t.shape[1]:2, 64:].copy_(t) for t in (p.q, p.k, p.v)]
    for q, k, v in (odd, turned, apart, [t.contiguous() for t in (p.q, p.k, p.v)]):
        assert torch.equal(packed_attention_hip(q, k, v, p.cu), want)
    assert torch.equal(packed_attention_hip(p.q, p.k, p.v, torch.stack((p.cu, p.cu), 1)[:, 0]), want)
    out = torch.zeros(rows, 4, 128, dtype=BF16, device="cuda")[..., 64:]
    assert torch.equal(p.attention(out=out), want)
    one = torch.zeros(1, 2, 64, dtype=BF16, device="cuda").expand(rows, 2, 64)  # one key for all rows
    assert not packed_attention_hip(p.q, one, one, p.cu).any()
    for bad in (p.q, p.k.expand(rows, 2, 64)):
        with pytest.raises(ValueError):
            packed_attention_hip(p.q, p.k, p.v, p.cu, out=bad)
    whole = torch.zeros(rows, 16, 64, dtype=BF16, device="cuda")  # output beside its inputs in one buffer
    whole[:, :4], whole[:, 4:6], whole[:, 6:8] = p.q, p.k, p.v
    assert torch.equal(packed_attention_hip(whole[:, :4], whole[:, 4:6], whole[:, 6:8], p.cu, out=whole[:, 8:12]), want)
    with pytest.raises(ValueError, match="share no memory"):
        packed_attention_hip(whole[:, :4], whole[:, 4:6], whole[:, 6:8], p.cu, out=whole[:, 6:10])


@gpu
def test_attention_refuses_on_the_gpu():
    p = Prompts([5])
    with pytest.raises(ValueError, match="head_dim of 64 or 128"):
        packed_attention_hip(p.q[..., :48].contiguous(), p.k[..., :48].contiguous(), p.v[..., :48].contiguous(), p.cu)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        packed_attention_hip(p.q[:, :3].contiguous(), p.k, p.v, p.cu)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        packed_attention_hip(p.q, p.k[:, :0], p.v[:, :0], p.cu)
    with pytest.raises(ValueError, match="finite"):
        p.attention(scale=math.inf)
    with pytest.raises(ValueError, match="must be a GPU tensor"):
        packed_attention_hip(p.q, p.k, p.v, p.cu.cpu())
    if torch.cuda.device_count() > 1:
        with pytest.raises(ValueError, match="same device"):
            packed_attention_hip(p.q, p.k.to("cuda:1"), p.v, p.cu)
    with torch.inference_mode(), pytest.raises(RuntimeError, match="function transform"):
        torch.vmap(lambda q: packed_attention_hip(q, p.k, p.v, p.cu))(p.q.unsqueeze(0))


@gpu
def test_attention_of_nothing():
    p = Prompts([0, 0])
    assert p.attention().shape == (0, 4, 64)
    q = Prompts([3])
    got = packed_attention_hip(q.q, q.k, q.v, ints([0]))
    assert got.shape == q.q.shape and not got.any()


@gpu
def test_rows_past_32_bit_offsets():
    """Rows so far apart that the last ones lie past 2^31 elements."""
    rows, stride = 150, 1 << 24
    base = torch.empty(rows * stride, dtype=BF16, device="cuda")
    p = Prompts([rows], heads=4, kv_heads=2, dim=64)
    wide = torch.as_strided(base, (rows, 8, 64), (stride, 64, 1))
    wide[:, :4], wide[:, 4:6], wide[:, 6:] = p.q, p.k, p.v
    assert torch.equal(packed_attention_hip(wide[:, :4], wide[:, 4:6], wide[:, 6:], p.cu), p.attention())
    out = torch.as_strided(base, (rows, 4, 64), (stride, 64, 1), 1024)
    p.attention(out=out)
    assert torch.equal(out, p.attention())


@gpu
def test_attention_repeats_bit_for_bit_and_on_other_streams():
    p = Prompts([700, 31, 90], heads=12, dim=128)
    want = p.attention()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [p.attention() for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(t, want) for t in others) and torch.equal(p.attention(), want)


@gpu
@pytest.mark.parametrize("lengths", [[40, 3, 120], [900], [300] * 30])
def test_attention_in_a_graph_with_other_lengths(lengths):
    """Captured once; the bounds and inputs change between replays, with eager work between."""
    p = Prompts(lengths, heads=12, dim=128)
    p.attention()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = p.attention()
    for turn in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, p.attention())
        near(out, *p.reference())
        p.v.copy_(torch.randn(p.v.shape, generator=p.gen, device="cuda"))
        b = turn % len(lengths)  # the sequence's last row goes to nobody, or to the next one
        p.lengths = [n - (i == b) + (i == b + 1) for i, n in enumerate(p.lengths)]
        p.cu.copy_(ints([sum(p.lengths[:i]) for i in range(len(lengths) + 1)]))


# ---------------------------------------------------------------------------
# Pages on the GPU
# ---------------------------------------------------------------------------

def _lists(*tensors):
    return tuple(t.tolist() for t in tensors)


class Pool:
    def __init__(self, seed, batch, width, pages, page, *, layers=2, heads=2, dim=64, dtype=BF16, token_major=False, flat=False,
                 spare=None, wild=False):
        self.page, spare = page, min(pages // 7, 9) if spare is None else spare
        self.table, self.lengths, self.users = state_of(seed, batch, width, pages, page, spare=spare, wild=wild)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        shape = (layers, pages, page, heads, dim) if token_major else (layers, pages, heads, page, dim)
        self.k, self.v = (torch.randn(shape, generator=gen, device="cuda").to(dtype) for _ in range(2))
        if token_major:
            self.k, self.v = self.k.transpose(2, 3), self.v.transpose(2, 3)
        if flat:
            self.k, self.v = self.k[0], self.v[0]

    def indices(self):
        return ints(self.table).view(len(self.table), -1), ints(self.lengths), ints(self.users)


@gpu
@pytest.mark.parametrize("wild", [False, True])
@pytest.mark.parametrize("sizes", POOLS + [(300, 40, 5000, 16), (9, 5000, 70000, 32), (1100, 7, 3000, 16)])
def test_resize_is_the_definition(sizes, wild):
    p = Pool(3, *sizes, layers=1, heads=1, dim=8, wild=wild)
    batch, width, pages, page = sizes
    gen = torch.Generator().manual_seed(1)
    table, _, users = p.indices()
    kept = table.clone(), users.clone()
    for wanted in (p.lengths, [0] * batch, [width * page] * batch,
                   torch.randint(0, width * page + 20, (batch,), generator=gen).tolist()):
        assert _lists(*paged_resize_hip(table, ints(wanted), users, page_size=page)) == resized(p.table, wanted, p.users, page)
    assert torch.equal(table, kept[0]) and torch.equal(users, kept[1])


@gpu
def test_resize_of_strided_tables_and_of_nothing():
    p = Pool(4, 7, 9, 70, 32, layers=1, heads=1, dim=8)
    table, lengths, users = p.indices()
    want = resized(p.table, p.lengths, p.users, 32)
    wide = torch.stack((table, table), 2).flatten(1)
    for t in (wide[:, ::2], torch.cat((table, table), 1)[:, :9]):
        assert _lists(*paged_resize_hip(t, torch.stack((lengths, lengths), 1)[:, 0], torch.stack((users, users), 1)[:, 1],
                                        page_size=32)) == want
    got = paged_resize_hip(table[:0], lengths[:0], users, page_size=32)
    assert got[0].shape == (0, 9) and torch.equal(got[1], users) and got[2].shape == (0,)
    big = torch.zeros(70000, dtype=I32, device="cuda")
    assert torch.equal(paged_resize_hip(table[:0], lengths[:0], big, page_size=32)[1], big)
    with pytest.raises(ValueError, match="power of two"):
        paged_resize_hip(table, lengths, users, page_size=24)
    with pytest.raises(ValueError, match="power of two"):
        paged_resize_hip(table, lengths, users, page_size=8)


@gpu
@pytest.mark.parametrize("wild", [False, True])
@pytest.mark.parametrize("sizes, more", [(sizes, {}) for sizes in POOLS] + [
    ((20, 70, 700, 16), {"token_major": True}), ((20, 70, 700, 16), {"flat": True, "dtype": F16, "dim": 128}),
    ((6, 3, 40, 64), {"layers": 5, "heads": 3, "dim": 72, "token_major": True}), ((3, 600, 70000, 16), {"layers": 1, "heads": 1}),
    ((1, 2, 9, 1024), {"heads": 8, "dim": 128}), ((700, 2, 3000, 16), {"layers": 1, "dim": 8}),
    ((30, 1200, 9000, 16), {"layers": 1, "dim": 8})])
def test_fork_is_the_definition(sizes, more, wild):
    batch, width, pages, page = sizes
    gen = torch.Generator().manual_seed(2)
    for parents in (list(range(batch)), [0] * 5, [], torch.randint(-1, batch + 1, (2 * batch,), generator=gen).tolist(),
                    [2 ** 31 - 1, -(2 ** 31), batch, -1]):
        p = Pool(5, *sizes, wild=wild, **more)
        want_k, want_v = p.k.clone(), p.v.clone()
        table, lengths, users = p.indices()
        kept = table.clone(), lengths.clone(), users.clone()
        got = paged_fork_hip(p.k, p.v, table, lengths, users, ints(parents))
        *want, copies = forked(p.table, p.lengths, p.users, parents, page)
        assert got[0].shape == (len(parents), width)
        assert _lists(*got) == tuple(want)
        for source, target, count in copies:
            for pool in (want_k, want_v):
                pool = pool if pool.dim() == 5 else pool.unsqueeze(0)
                pool[:, target, :, :count] = pool[:, source, :, :count]
        assert torch.equal(p.k, want_k) and torch.equal(p.v, want_v)
        assert all(torch.equal(a, b) for a, b in zip((table, lengths, users), kept))


@gpu
@pytest.mark.parametrize("wild", [False, True])
@pytest.mark.parametrize("sizes, more", [(sizes, {}) for sizes in POOLS] + [
    ((20, 70, 700, 16), {"token_major": True}), ((20, 70, 700, 16), {"flat": True, "dtype": F16, "dim": 128}),
    ((6, 3, 40, 64), {"layers": 5, "heads": 3, "dim": 72, "token_major": True}), ((3, 600, 70000, 16), {"layers": 1, "heads": 1}),
    ((1, 2, 9, 1024), {"heads": 8, "dim": 128}), ((1100, 2, 3000, 16), {"layers": 1, "dim": 8}),
    ((30, 1200, 9000, 16), {"layers": 1, "dim": 8}), ((1100, 2, 17000, 16), {"layers": 1, "heads": 1, "dim": 8}),
    ((700, 800, 3000, 16), {"layers": 1, "heads": 1, "dim": 8})])
def test_compact_is_the_definition(sizes, more, wild):
    batch, width, pages, page = sizes
    for turn in range(6):
        p = Pool(6, *sizes, wild=wild, **more)
        counts = (p.users, [0] * pages, [1] * pages, [n if i % 3 else 0 for i, n in enumerate(p.users)],
                  [int(i >= pages // 2) for i in range(pages)], [2 * int(i < pages // 2) for i in range(pages)])[turn]
        table, _, _ = p.indices()
        users = ints(counts)
        before = p.k.clone(), p.v.clone()
        got = paged_compact_hip(p.k, p.v, table, users)
        want = compacted(p.table, counts)
        assert _lists(*got) == want
        to = torch.tensor(want[2], device="cuda")
        source = torch.arange(pages, device="cuda")
        source[to[to >= 0]] = (to >= 0).nonzero().view(-1)
        live = int((to >= 0).sum())
        for pool, old in zip((p.k, p.v), before):
            pool, old = (t if t.dim() == 5 else t.unsqueeze(0) for t in (pool, old))
            assert torch.equal(pool[:, :live], old[:, source[:live]]) and torch.equal(pool[:, live:], old[:, live:])


@gpu
def test_copies_of_pages_past_32_bit_offsets():
    """A pool of more than 2^31 elements; its last pages move and are forked."""
    pages, page, heads, dim = 131080 + 16, 64, 2, 128
    pools = [torch.empty(pages, heads, page, dim, dtype=BF16, device="cuda") for _ in range(2)]
    users = torch.zeros(pages, dtype=I32, device="cuda")
    users[[pages - 1, pages - 3]] = 1
    gen = torch.Generator(device="cuda").manual_seed(3)
    small = [torch.randn(2, heads, page, dim, generator=gen, device="cuda").to(BF16) for _ in range(2)]
    for pool, part in zip(pools, small):
        pool[[pages - 3, pages - 1]] = part
    table = ints([[pages - 1, -1], [pages - 3, -1]])
    new, lengths, after, missing = paged_fork_hip(*pools, table, ints([50, 64]), users, ints([0, 0, 1, 1]))
    assert new.tolist() == [[pages - 1, -1], [0, -1], [pages - 3, -1], [pages - 3, -1]] and not missing.any()
    for pool, part in zip(pools, small):
        assert torch.equal(pool[0, :, :50], part[1, :, :50])
    last = torch.zeros(pages, dtype=I32, device="cuda")
    last[:-4] = 1  # (a copy whose target lies far behind)
    last[pages - 1] = 1
    for pool in pools:
        pool[0] = pool[pages - 1]
    new, _, _, _ = paged_fork_hip(*pools, ints([[0], [pages - 1]]), ints([20, 3]), last, ints([0, 0]))
    assert new.tolist() == [[0], [pages - 4]]
    for pool, part in zip(pools, small):
        assert torch.equal(pool[pages - 4, :, :20], part[1, :, :20])
    users = torch.zeros(pages, dtype=I32, device="cuda")
    users[[pages - 1, pages - 3]] = 1
    new, after, to = paged_compact_hip(*pools, table, users)
    assert new.tolist() == [[1, -1], [0, -1]] and after[:3].tolist() == [1, 1, 0]
    for pool, part in zip(pools, small):
        assert torch.equal(pool[:2], part)


@gpu
def test_page_operators_in_one_graph():
    """Resize, fork and compact captured together; each replay starts from the state that the
    last one left, with eager work between."""
    p = Pool(7, 12, 9, 150, 16, layers=3)
    table, lengths, users = p.indices()
    wanted, parents = lengths.clone(), ints(list(range(12)))
    state = [t.clone() for t in (table, lengths, users)]
    pools = p.k.clone(), p.v.clone()

    def step(table, lengths, users, k, v):
        t, u, missing = paged_resize_hip(table, wanted, users, page_size=16)
        t, n, u, lacks = paged_fork_hip(k, v, t, wanted, u, parents)
        t, u, to = paged_compact_hip(k, v, t, u)
        return t, n, u, missing, lacks, to

    step(*state, *pools)
    for a, b in zip(pools, (p.k, p.v)):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        answers = step(table, lengths, users, p.k, p.v)
        table.copy_(answers[0])
        lengths.copy_(answers[1])
        users.copy_(answers[2])
    gen = torch.Generator().manual_seed(9)
    for turn in range(5):
        wanted.copy_(torch.randint(0, 9 * 16 + 1, (12,), generator=gen))
        parents.copy_(torch.randint(-1, 12, (12,), generator=gen))
        want = step(*state, *pools)
        state = [t.clone() for t in want[:3]]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(answers, want))
        assert torch.equal(p.k, pools[0]) and torch.equal(p.v, pools[1])


@gpu
def test_many_children_of_one_row():
    """More of them than free pages: the last ones lack theirs."""
    p = Pool(1, 2, 3, 1500, 16, layers=1, heads=1, dim=8)
    p.table, p.lengths = [[0, 1, -1], [2, -1, -1]], [20, 16]
    p.users = [1, 1, 1] + [0] * 1400 + [1] * 97
    for children in (900, 1700):
        parents = [0] * children + [1, 1]
        k = p.k.clone()
        got = paged_fork_hip(k, p.v.clone(), *p.indices(), ints(parents))
        *want, copies = forked(p.table, p.lengths, p.users, parents, 16)
        assert _lists(*got) == tuple(want) and sum(want[3]) == max(0, children - 1401)
        for source, target, count in copies:
            assert torch.equal(k[:, target, :, :count], p.k[:, source, :, :count])
            assert torch.equal(k[:, target, :, count:], p.k[:, target, :, count:])


@gpu
@pytest.mark.parametrize("spare", [0, 2000])
@pytest.mark.parametrize("batch, width, pages", [(50, 4, 2000), (1500, 3, 6000), (3, 300, 40000)])
def test_more_children_than_a_workgroup_has_threads(batch, width, pages, spare):
    """Copies are counted by parts of the children; without spare pages some find none."""
    page = 16
    p = Pool(8, batch, width, pages, page, layers=1, heads=1, dim=8, spare=spare and pages // 4)
    table, lengths, users = p.indices()
    gen = torch.Generator().manual_seed(4)
    for parents in (torch.randint(-1, batch + 1, (5000,), generator=gen).tolist(), [batch - 1] * 2049,
                    [i // 3 if i % 64 else -1 for i in range(3 * batch)]):
        want_k, want_v = p.k.clone(), p.v.clone()
        k, v = p.k.clone(), p.v.clone()
        got = paged_fork_hip(k, v, table, lengths, users, ints(parents))
        *want, copies = forked(p.table, p.lengths, p.users, parents, page)
        assert _lists(*got) == tuple(want)
        for source, target, count in copies:
            want_k[:, target, :, :count] = want_k[:, source, :, :count]
            want_v[:, target, :, :count] = want_v[:, source, :, :count]
        assert torch.equal(k, want_k) and torch.equal(v, want_v)


@gpu
def test_page_operators_on_other_streams_and_side_by_side():
    """Keys and values in one buffer; calls on two streams at once; indices in strides."""
    p = Pool(2, 20, 70, 700, 16, layers=3, token_major=True)
    both = torch.stack((p.k, p.v), 1)
    k, v = both.unbind(1)
    table, lengths, users = p.indices()
    parents = list(range(20)) + [3, 3, 7]
    *want, copies = forked(p.table, p.lengths, p.users, parents, 16)
    other = resized(p.table, [9] * 20, p.users, 16)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    wide = torch.stack((table, table), 2)[:, :, 1]
    for stream in (a, b):
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(a):
            got = paged_fork_hip(k, v, wide, lengths, users, ints(parents))
        with torch.cuda.stream(b):
            cut = paged_resize_hip(table, ints([9] * 20), users, page_size=16)
            cut_too = paged_resize_hip(table.expand(1, 20, 70)[0], ints([9] * 20), users, page_size=16)
        torch.cuda.synchronize()
        assert _lists(*got) == tuple(want) and _lists(*cut) == other and _lists(*cut_too) == other
    for source, target, count in copies:
        assert torch.equal(both[:, :, target, :, :count], both[:, :, source, :, :count])
    with torch.inference_mode():
        assert _lists(*paged_resize_hip(table, ints([9] * 20), users, page_size=16)) == other


@gpu
def test_two_captured_graphs_share_no_workspace():
    """Replayed in turn and side by side, each gives its own answer."""
    a, b = Pool(8, 300, 60, 4000, 16, layers=1, heads=1, dim=8), Pool(9, 300, 60, 4000, 16, layers=1, heads=1, dim=8)
    calls = []
    for p in (a, b):
        t = p.indices()
        paged_resize_hip(*t, page_size=16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = paged_resize_hip(*t, page_size=16)
        calls.append((graph, got, resized(p.table, p.lengths, p.users, 16), torch.cuda.Stream(), t))  # (t stays alive)
    for turn in range(3):
        for graph, _, _, stream, _ in calls:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, got, want, _, _ in calls:
            assert _lists(*got) == want


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_serving_with_pages_end_to_end(dtype):
    """Two prompts of unequal length: pages given out, rows appended, the prompts attended where
    they stand; then both forked, each fork continued by a token of its own, the first ended,
    the pool compacted.  What the forks attend over the pages is the formula's over their
    whole histories."""
    heads, kv_heads, dim, page = 4, 2, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(0)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    k_pages, v_pages = (torch.full((40, kv_heads, page, dim), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    users, table = torch.zeros(40, dtype=I32, device="cuda"), torch.full((2, 8), -1, dtype=I32, device="cuda")
    inv = torch.rand(dim // 2, device="cuda")
    lengths, cu = ints([37, 16]), ints([0, 37, 53])
    table, users, missing = paged_resize_hip(table, lengths, users, page_size=page)
    assert not missing.any() and int(users.sum()) == 4
    qkv = randn(53, heads + 2 * kv_heads, dim)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
    rotated = paged_append_hip(qkv[:, :heads + kv_heads], k, v, k_pages, v_pages, table, cu, lengths, inv)
    got = packed_attention_hip(rotated[:, :heads], rotated[:, heads:], v, cu)
    p = Prompts([37, 16], heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    p.q, p.k, p.v = rotated[:, :heads], rotated[:, heads:], v
    near(got, *p.reference())
    # the same rows through the pages: within a half step of the output and of each probability
    paged = paged_attention_hip(rotated[:, :heads], k_pages, v_pages, table, cu, lengths)
    assert float((paged.double() - got.double()).abs().amax()) < 4 * torch.finfo(dtype).eps
    history = [(rotated[:37, heads:], v[:37]), (rotated[37:, heads:], v[37:])]
    parents = [0, 1, 0, 0]
    table, lengths, users, missing = paged_fork_hip(k_pages, v_pages, table, lengths, users, ints(parents))
    assert lengths.tolist() == [37, 16, 37, 37] and not missing.any()
    assert sorted(users.tolist(), reverse=True)[:6] == [3, 3, 1, 1, 1, 1]
    lengths = lengths + 1
    table, users, missing = paged_resize_hip(table, lengths, users, page_size=page)
    qkv, cu = randn(4, heads + 2 * kv_heads, dim), ints([0, 1, 2, 3, 4])
    rotated = paged_append_hip(qkv[:, :heads + kv_heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], k_pages, v_pages,
                               table, cu, lengths, inv)
    lengths[0] = 0
    table, users, missing = paged_resize_hip(table, lengths, users, page_size=page)
    table, users, to = paged_compact_hip(k_pages, v_pages, table, users)
    live = int((users > 0).sum())
    assert live == 2 + 1 + 1 + 2 and bool((table[0] == -1).all()) and int((to >= 0).sum()) == live
    got = paged_attention_hip(rotated[:, :heads], k_pages[:live], v_pages[:live], table, cu, lengths)
    assert not got[0].any()
    for row, parent in list(enumerate(parents))[1:]:
        keys, values = (torch.cat((old, new[row:row + 1]))
                        for old, new in zip(history[parent], (rotated[:, heads:], qkv[:, heads + kv_heads:])))
        for h in range(heads):
            g = h // 2
            w = torch.softmax(keys[:, g].double() @ rotated[row, h].double() * dim ** -0.5, 0)
            want = w @ values[:, g].double()
            assert float((got[row, h].double() - want).abs().amax()) < 2 * torch.finfo(dtype).eps


def test_every_operator_is_named():
    for name in ("packed_attention_hip", "paged_resize_hip", "paged_fork_hip", "paged_compact_hip"):
        assert name in qwen_int4_hip.__all__ and getattr(qwen_int4_hip, name).__doc__
