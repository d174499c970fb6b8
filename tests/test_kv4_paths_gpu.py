"""Attention over a cache in 4 bits: which path a request takes, and that path's own bound against 64 bits (tests/plain_kv4_bounds.py)."""
import pytest
import torch

import plain_kv4_bounds as bounds
from mini_sglang_b200 import ops
from mini_sglang_b200.parts import Workspace
from test_kv4_edges_gpu import attend, table_of
from test_kv4_gpu import BF, F32, GEOMETRIES, filled, i32, normal

pytestmark = pytest.mark.gpu


class Library:
    """The built library, noting which entry points are called."""

    def __init__(self, lib, log):
        self.lib, self.log = lib, log

    def __getattr__(self, name):
        f = getattr(self.lib, name)
        return lambda *a: self.log.append(name) or f(*a)


def run(monkeypatch, q_lens, kv_lens, n_q, n_kv, d, dtype, page=16, window=0, seed=0, host=True):
    """(result, 64 bits, bound of either path, entry points called)."""
    width = -(-max(kv_lens) // page)
    table = (torch.randperm(len(kv_lens) * width, generator=torch.Generator().manual_seed(seed)) + 1).view(-1, width).int().cuda()
    c, q = filled(seed + 3, table.numel() + 1, n_kv, page, d), normal(seed + 5, sum(q_lens), n_q, d, dtype=dtype)
    starts, log, lib = [sum(q_lens[:i]) for i in range(len(q_lens) + 1)], [], ops._kv4_lib()
    with monkeypatch.context() as m:
        m.setattr(ops, "_kv4_lib", lambda: Library(lib, log))
        out = attend(q, c, kv_lens, table, window=window, workspace=Workspace("cuda"), **(dict(q_start=i32(starts), q_lens=q_lens, kv_lens=kv_lens) if host else {}))
    ops.check_kernel_status()
    direct = "codes" if dtype == BF and d in (64, 128) else "float32"
    want, off = bounds.attention(q, c, starts, q_lens, kv_lens, table, d ** -0.5, window, direct)
    restored = bounds.attention(q, c, starts, q_lens, kv_lens, table, d ** -0.5, window, "restored" if dtype == BF else "float32")[1]
    return out, want, off, restored, log


def inside(out, want, off):
    assert ((out.double() - want).abs() <= off + torch.finfo(out.dtype).eps / 2 * (want.abs() + off)).all()


def direct(out, want, off, log):
    assert set(log) <= {"msgl_kv4_attention_runs", "msgl_kv4_attention_any"} and log
    inside(out, want, off)
    # Normal values and many results: rounding to bfloat16 leaves errors of 2^-8 / sqrt(3) / 1.47 = 1.5e-3 of their size (1.47: the root of the mean square of a mantissa spread evenly
    # over its logarithm), weights rounded to 2^-11 of themselves 0.4 * 2.6 * 2^-11 = 0.5e-3 (2.6: 7.5 codes of 0.35 of a deviation), together below 2^-9.  Restored keys give twice that.
    if out.numel() >= 2048:
        assert (out.double() - want).norm() <= (2.0 ** -9 if out.dtype == BF else 2.0 ** -18) * want.norm()


@pytest.mark.parametrize("n_q,n_kv,d,dtype", GEOMETRIES)
@pytest.mark.parametrize("kv_lens", [[1], [5, 64, 1, 129], [700, 31, 32, 33], [2049] * 3])
@pytest.mark.parametrize("host", [False, True])
def test_single_tokens_read_codes(monkeypatch, n_q, n_kv, d, dtype, kv_lens, host):
    out, want, off, _, log = run(monkeypatch, [1] * len(kv_lens), kv_lens, n_q, n_kv, d, dtype, host=host)
    direct(out, want, off, log)


@pytest.mark.parametrize("n_q,n_kv,d,dtype", GEOMETRIES)
@pytest.mark.parametrize("window", [0, 33])
def test_a_few_tokens_read_codes(monkeypatch, n_q, n_kv, d, dtype, window):
    out, want, off, _, log = run(monkeypatch, [3, 1, 2, 2], [3, 300, 137, 800], n_q, n_kv, d, dtype, window=window, page=8, seed=1)
    if 3 * n_q // n_kv <= (80 if dtype == BF and d in (64, 128) else 32):
        direct(out, want, off, log)


@pytest.mark.parametrize("n_q,n_kv,d,dtype", [(8, 2, 128, BF), (32, 8, 128, BF), (4, 2, 64, BF), (4, 4, 40, BF), (4, 2, 128, F32), (3, 1, 40, F32)])
@pytest.mark.parametrize("window", [0, 100])
def test_portions_are_restored_and_single_tokens_beside_them_are_not(monkeypatch, n_q, n_kv, d, dtype, window):
    monkeypatch.setattr(ops, "_kv4_middle", lambda q_lens, kv_lens, direct, *a: direct)
    lens, kv = [150, 1, 90, 2, 1], [200, 700, 90, 333, 31]
    out, want, off, restored, log = run(monkeypatch, lens, kv, n_q, n_kv, d, dtype, window=window, seed=2)
    assert log.count("msgl_kv4_restore") == 1 and len(log) == 2
    few = torch.zeros(sum(lens), dtype=torch.bool, device="cuda")
    for r in (1, 3, 4):
        few[sum(lens[:r]):sum(lens[:r + 1])] = True
    inside(out[few], want[few], off[few])
    inside(out[~few], want[~few], restored[~few])
    # restored keys, values and weights are each rounded to 2^-8 of themselves, as the result is: each at most what direct() says of the result, a score's errors about as much again
    assert (out[~few].double() - want[~few]).norm() <= (2.0 ** -7 if dtype == BF else 2.0 ** -18) * want[~few].norm()


@pytest.mark.parametrize("page", [1, 16, 48, 256])
@pytest.mark.parametrize("window", [0, 1, 50])
@pytest.mark.parametrize("d", [64, 128])
def test_pages_and_windows_from_codes(monkeypatch, page, window, d):
    out, want, off, _, log = run(monkeypatch, [1, 6, 1, 4], [333, 90, 12, 280], 8, 2, d, BF, page=page, window=window, seed=page)
    direct(out, want, off, log)
