"""The paged kernels' own sources compiled for the CPU (tests/lanes), every buffer in
a mapping of its own with nothing mapped around it: an access outside a buffer ends
the process, at lengths and row bounds that need no GPU to be tried.  Each check runs
in a process of its own, once with its buffers against their mappings' ends and once
against their starts."""

from __future__ import annotations

import ctypes
import math
import re
import subprocess
import sys
from pathlib import Path

import pytest
import torch

REPO = Path(__file__).resolve().parents[1]
CSRC = REPO / "qwen2-int4-systems_amd" / "csrc"
LANES = Path(__file__).resolve().parent / "lanes"
SOURCES = ("qwen2_paged_append", "qwen2_paged_attention", "qwen2_verify")
BF16 = torch.bfloat16

INTERNAL = """
#pragma once
#include <hip/hip_runtime.h>
#include "w4g64.h"
namespace w4g64 {
constexpr int kAttnHeadDim = 128;
int set_error(int status, const char* fmt, ...);
int clear_error();
}
"""


def _compiler():
    from qwen_int4_hip import build

    clang = Path(build.hipcc()).resolve().parents[1] / "llvm" / "bin" / "clang++"
    if not clang.exists():
        pytest.skip(f"no compiler for the CPU at {clang}")
    return clang


@pytest.fixture(scope="module")
def lanes_library(tmp_path_factory):
    root = tmp_path_factory.mktemp("lanes")
    for path in [*CSRC.glob("*.h"), *(CSRC / f"{name}.hip" for name in SOURCES)]:
        text = path.read_text()
        # (GPU registers and address spaces are the only words of the language that the CPU lacks)
        text = re.sub(r'asm volatile\("" : "\+[sv]"\((\w)\)\);', r'asm volatile("" : "+r"(\1));', text)
        text = re.sub(r"__attribute__\(\(address_space\(\d+\)\)\)", "", text)
        (root / path.name).write_text(text)
    (root / "w4g64_internal.h").write_text(INTERNAL)
    flags = ["-std=c++17", "-O2", "-fPIC", "-ffp-contract=off", "-mf16c", "-mfma", "-w", f"-I{LANES}", f"-I{root}",
             f"-I{REPO / 'include'}"]
    compiler = _compiler()
    jobs = [subprocess.Popen([compiler, *flags, "-x", "c++", "-c", str(source), "-o", str(root / f"{source.stem}.o")],
                             stderr=subprocess.PIPE, text=True)
            for source in [LANES / "lanes.cpp", *(root / f"{name}.hip" for name in SOURCES)]]
    for job in jobs:
        said = job.communicate()[1]
        assert job.returncode == 0, said
    library = root / "lanes.so"
    subprocess.run([compiler, "-shared", *map(str, root.glob("*.o")), "-o", str(library)], check=True)
    return library


# ---------------------------------------------------------------------------
# In the process of a check
# ---------------------------------------------------------------------------

class Memory:
    """Tensors in mappings of their own."""

    def __init__(self, side):
        self.side, self.libc = side, ctypes.CDLL(None)
        self.libc.mmap.restype = ctypes.c_void_p
        self.libc.mmap.argtypes = [ctypes.c_void_p, ctypes.c_size_t] + [ctypes.c_int] * 3 + [ctypes.c_long]
        self.libc.mprotect.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]

    def __call__(self, t):
        count, gap = max(t.numel() * t.element_size(), 1), 16 << 20
        inner = -(-count // 4096) * 4096
        base = self.libc.mmap(None, inner + 2 * gap, 0, 0x22, -1, 0)  # private, of nothing, no access
        assert base and self.libc.mprotect(base + gap, inner, 3) == 0
        # (to an alignment of 16 bytes: what ends short of it has a gap of less)
        at = base + gap + ((inner - count) // 16 * 16 if self.side == "end" else 0)
        return torch.frombuffer((ctypes.c_ubyte * count).from_address(at), dtype=t.dtype)[:t.numel()].view(t.shape).copy_(t)


class Kernels:
    def __init__(self, library, side):
        from qwen_int4_hip import _lib

        self.abi, self.memory, self.lib = _lib, Memory(side), ctypes.CDLL(library)
        for name in ("qwen2_paged_append", "qwen2_paged_attention_workspace_bytes", "qwen2_paged_attention",
                     "qwen2_verify_drafts_workspace_bytes", "qwen2_verify_drafts"):
            getattr(self.lib, name).restype, getattr(self.lib, name).argtypes = _lib.SIGNATURES[name]
        self.lib.lanes_error.restype = ctypes.c_char_p

    def check(self, status):
        assert status == 0, (status, self.lib.lanes_error())

    def rows(self, t):
        return ctypes.byref(self.abi.Rows(t.data_ptr(), t.stride(0), t.stride(1)))

    def cache(self, k, v, table, cu, lengths):
        return ctypes.byref(self.abi.PagedCache(
            k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], k.shape[0], k.shape[2], table.data_ptr(),
            table.shape[1], table.stride(0), cu.data_ptr(), lengths.data_ptr(), table.shape[0], k.shape[1], k.shape[3],
            {torch.float16: 1, BF16: 2}[k.dtype]))

    def attention(self, q, k, v, table, cu, lengths, shared, zero_rest=1, fill=0.0):
        out, cache = self.memory(torch.full_like(q, fill)), self.cache(k, v, table, cu, lengths)
        need = self.lib.qwen2_paged_attention_workspace_bytes(cache, q.shape[0], q.shape[1], shared)
        workspace = self.memory(torch.full((need,), 0xA5, dtype=torch.uint8))
        self.check(self.lib.qwen2_paged_attention(cache, self.rows(q), self.rows(out), q.shape[0], q.shape[1], shared,
                                                  q.shape[2] ** -0.5, zero_rest, workspace.data_ptr(), need, None))
        return out, need


def _batch(kernels, *, batch, rows, heads, kv_heads, dim, page, shared, past, tail=0, dtype=BF16):
    """Sequences of equal length: (q, k, v, table, cu, lengths) of a call."""
    gen = torch.Generator().manual_seed(rows + past)
    own = -(-(rows + past) // page)
    order = torch.randperm(shared + batch * own, generator=gen).to(torch.int32)
    table = torch.cat((order[:shared].expand(batch, shared), order[shared:].view(batch, own)), 1)
    k, v = (torch.randn(len(order), kv_heads, page, dim, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(batch * rows + tail, heads, dim, generator=gen).to(dtype)
    cu = torch.arange(batch + 1, dtype=torch.int32) * rows
    lengths = torch.full((batch,), shared * page + rows + past, dtype=torch.int32)
    return [kernels.memory(t) for t in (q, k, v, table, cu, lengths)]


def _formula(q, k, v, table, cu, lengths):
    """Attended rows in 64 bits."""
    out, page, group = torch.zeros(q.shape, dtype=torch.float64), k.shape[2], q.shape[1] // k.shape[1]
    for b in range(len(lengths)):
        first, end, length = int(cu[b]), int(cu[b + 1]), int(lengths[b])
        at = torch.arange(length)
        keys, values = (c[table[b].long()[at // page], :, at % page].double() for c in (k, v))
        for r in range(first, end):
            sees = length - (end - first) + (r - first) + 1
            for h in range(q.shape[1]):
                w = torch.softmax(keys[:sees, h // group] @ q[r, h].double() * q.shape[2] ** -0.5, 0)
                out[r, h] = w @ values[:sees, h // group]
    return out


FAR = {  # the largest contexts of the calls, both ends of the page table in use
    "64x5 over 16384": dict(batch=64, rows=5, heads=12, kv_heads=2, dim=128, page=64, shared=256, past=0),
    "16x5 over 65536": dict(batch=16, rows=5, heads=6, kv_heads=1, dim=128, page=64, shared=1024, past=0),
    "16x5 over 32768": dict(batch=16, rows=5, heads=6, kv_heads=1, dim=128, page=64, shared=512, past=0),
    "1x1 after 131071": dict(batch=1, rows=1, heads=12, kv_heads=2, dim=128, page=64, shared=0, past=131071),
}


def _far(kernels, name):
    kernels.lib.lanes_skip_products(1)  # (which addresses are used does not depend on them)
    out, _ = kernels.attention(*_batch(kernels, **FAR[name]), FAR[name]["shared"])
    assert bool(out.isfinite().all())


def _small(kernels, name):
    """Outputs of both forms and of the join against 64 bits; then infinities among the
    values, so that sums are counted anew: what is expected is that rows which see them
    are not finite and the others are."""
    for case in (dict(batch=2, rows=3, past=70, shared=3, heads=4, kv_heads=2, dim=64, page=16),
                 dict(batch=2, rows=30, past=40, shared=5, heads=12, kv_heads=2, dim=64, page=32),
                 dict(batch=1, rows=1, past=300, shared=0, heads=2, kv_heads=1, dim=128, page=16, dtype=torch.float16)):
        args = _batch(kernels, **case)
        out, _ = kernels.attention(*args, case["shared"])
        # (16-bit rounding of the output; probabilities to 2^-17, values of a few units)
        assert float((out.double() - _formula(*args)).abs().amax()) < 4 * torch.finfo(out.dtype).eps
        q, k, v, table, cu, lengths = args
        last = int(lengths[0]) - 1
        v[int(table[0, last // case["page"]]), :, last % case["page"]] = math.inf
        out, _ = kernels.attention(*args, case["shared"])
        seen = case["rows"] - 1
        assert not out[seen].isfinite().any()
        out[seen] = 0
        assert bool(out.isfinite().all())


def _bounds(kernels, name):
    """Row bounds that fall or lead out, calls of one split and of several, own pages and
    none: no access outside the buffers, and rows behind the last bound as they were (or
    zeros)."""
    wild = [[0, 2, 2 ** 31 - 1], [0, 2 ** 31 - 1, -(2 ** 31)], [-7, 90, 2], [3, 1, 0], [0, 0, -1], [0, 3, 3],
            [2 ** 31 - 1] * 3, [-(2 ** 31)] * 3]
    for case in (dict(rows=2, past=30, shared=0), dict(rows=2, past=30, shared=2), dict(rows=2, past=300, shared=0),
                 dict(rows=70, past=9, shared=3)):
        q, k, v, table, _, lengths = args = _batch(kernels, batch=2, heads=4, kv_heads=2, dim=64, page=16, tail=3, **case)
        for values in wild:
            args[4] = cu = kernels.memory(torch.tensor(values, dtype=torch.int64).to(torch.int32))
            end = min(max(values[-1], 0), q.shape[0])
            for wrong in (lengths, kernels.memory(torch.tensor([2 ** 31 - 1, -(2 ** 31)]).to(torch.int32))):
                args[5] = wrong
                for width in (table.shape[1], max(case["shared"], 1)):
                    args[3] = kernels.memory(table[:, :width].contiguous())
                    for zero_rest in (0, 1):
                        out, need = kernels.attention(*args, case["shared"], zero_rest, fill=7.0)
                        assert bool((out[end:] == (0.0 if zero_rest else 7.0)).all()), (case, values, width, zero_rest, need)
            turned, inv = kernels.memory(torch.full_like(q, 7.0)), kernels.memory(torch.ones(32))
            new = [kernels.memory(torch.zeros(q.shape[0], 2, 64, dtype=BF16)) for _ in range(2)]
            pages = [kernels.memory(t) for t in (k, v)]
            kernels.check(kernels.lib.qwen2_paged_append(
                kernels.cache(*pages, table, cu, lengths), kernels.rows(q), *map(kernels.rows, new), kernels.rows(turned),
                inv.data_ptr(), 64, 0, 1.0, q.shape[0], 4, 0, None))
            assert bool((turned[end:] == 7.0).all())


def _verification(kernels, name):
    for dtype, code in ((torch.float32, 3), (BF16, 2)):
        for vocab in (1, 1001, 33000):
            gen = torch.Generator().manual_seed(vocab)
            p = kernels.memory(torch.softmax(torch.randn(3, 3, vocab, generator=gen), -1).to(dtype))
            d = kernels.memory(torch.softmax(torch.randn(3, 2, vocab, generator=gen), -1).to(dtype))
            ids = kernels.memory(torch.tensor([[0, vocab - 1], [vocab, -1], [2 ** 62, 0]]))
            counts, u = kernels.memory(torch.tensor([2, 2 ** 31 - 1, -(2 ** 31)]).to(torch.int32)), kernels.memory(torch.rand(3, 3, generator=gen))
            tokens, accepted = kernels.memory(torch.zeros(3, 3, dtype=torch.int64)), kernels.memory(torch.zeros(3, dtype=torch.int32))
            need = kernels.lib.qwen2_verify_drafts_workspace_bytes(3, 2, vocab)
            workspace = kernels.memory(torch.zeros(need, dtype=torch.uint8))
            for draft in (d, None):
                kernels.check(kernels.lib.qwen2_verify_drafts(
                    p.data_ptr(), *p.stride()[:2], draft.data_ptr() if draft is not None else None, *d.stride()[:2], code,
                    ids.data_ptr(), counts.data_ptr(), u.data_ptr(), tokens.data_ptr(), accepted.data_ptr(), 3, 2, vocab,
                    workspace.data_ptr(), need, None))
                new = tokens.gather(1, accepted.long().view(-1, 1))
                assert accepted[1:].tolist() == [0, 0] and bool(((new >= 0) & (new < vocab)).all())


CHECKS = {name: _far for name in FAR} | {"small": _small, "bounds": _bounds, "verification": _verification}


@pytest.mark.parametrize("side", ["end", "start"])
@pytest.mark.parametrize("name", CHECKS)
def test_every_access_lies_in_its_buffer(lanes_library, name, side):
    result = subprocess.run([sys.executable, __file__, str(lanes_library), name, side], capture_output=True, text=True,
                            timeout=300)
    assert result.returncode == 0 and result.stdout.endswith("done\n"), (result.returncode, result.stderr[-2000:])


if __name__ == "__main__":
    sys.path.insert(0, str(REPO / "qwen2-int4-systems_amd"))
    torch.set_num_threads(1)
    CHECKS[sys.argv[2]](Kernels(sys.argv[1], sys.argv[3]), sys.argv[2])
    print("done")
