"""Log probabilities of given tokens, entropies and top tokens against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
STEP = 2.0 ** -24          # half a step of float32 at one


def plain(logits, tokens, top):
    x = logits.double()
    lp = torch.log_softmax(x, 1)
    ok = (tokens >= 0) & (tokens < x.shape[1])
    given = torch.where(ok, lp.gather(1, tokens.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0], math.nan)
    entropy = -(lp.exp() * lp).nan_to_num(nan=0.0).sum(1)          # (0 x -inf counts nothing)
    entropy[lp.isnan().any(1)] = math.nan
    order = torch.sort(x.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf), dim=1, descending=True, stable=True).indices[:, :top]
    return given, entropy, lp.gather(1, order), order


def check(logits, tokens, top):
    from mini_sglang_b200 import ops
    got = ops.token_logprobs(logits, tokens, top)
    given, entropy, best, ids = plain(logits, tokens, top)
    V = logits.shape[1]
    # the sums have at most V / 256 terms one after the other in a thread and a few dozen joins, each off by half a step of the partial
    # sum, and exponentials off by four half steps and by the rounding of their argument, |x - m| half steps, of which those that weigh
    # have little; the difference x - m and the logarithm are rounded once each
    steps = V / 256 + 96
    for mine, want in ((got.logprobs, given), (got.top_logprobs, best)):
        assert torch.equal(mine.isnan(), want.isnan()) and torch.equal(mine.isinf(), want.isinf())
        fine = want.isfinite()
        assert ((mine.double() - want).abs()[fine] <= STEP * (steps + 4 * want.abs()[fine])).all()
    assert torch.equal(got.entropy.isnan(), entropy.isnan())
    fine = entropy.isfinite()
    # t / s has the errors of both sums, and entropy = log s - t / s
    assert ((got.entropy.double() - entropy).abs()[fine] <= STEP * (2 * steps * (1 + entropy[fine]) + 64)).all()
    if not logits.isnan().any():
        assert torch.equal(got.top_tokens.long(), ids)
    return got


SIZES = [(1, 1, 1), (1, 2, 2), (3, 7, 5), (2, 8, 8), (5, 31, 31), (4, 257, 20), (1, 32, 32), (7, 1000, 0), (1, 151936, 20), (64, 151936, 5), (700, 5000, 3),
         (2, 16383, 32), (2, 16385, 1), (3, 32003, 8), (40, 4097, 20), (1, 300001, 20)]


@pytest.mark.parametrize("rows,vocab,top", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_random_rows(rows, vocab, top, dtype):
    g = torch.Generator(device=DEV).manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=g, device=DEV) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV).to(torch.int32)
    check(logits, tokens, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_strided_rows(dtype, offset):
    """Rows that start anywhere and lie apart; what lies between them is not read."""
    g = torch.Generator(device=DEV).manual_seed(2)
    wide = torch.full((6, 5011), math.nan, device=DEV, dtype=dtype)
    wide[:, offset:offset + 4999] = torch.randn(6, 4999, generator=g, device=DEV).to(dtype)
    check(wide[:, offset:offset + 4999], torch.arange(6, device=DEV, dtype=torch.int32) * 800, 9)


def test_ties_and_orders():
    """Equal logits come by index, rising and falling rows are walked whole, zeros of both signs are equal."""
    V = 20011
    ramp = torch.arange(V, device=DEV, dtype=torch.float32)
    rows = torch.stack([torch.zeros(V, device=DEV), torch.full((V,), -3.5, device=DEV), ramp * 1e-3, -ramp * 1e-3, (ramp % 7) - 3, ramp.fmod(2) * -0.0,
                        torch.where(ramp % 2 == 0, 0.0, -0.0)])
    tokens = torch.tensor([0, V - 1, V - 1, 0, 3, 5, 6], dtype=torch.int32, device=DEV)
    for top in (1, 7, 20, 32):
        check(rows, tokens, top)


def test_masked_rows():
    """-inf counts for nothing, also where hardly anything else is left; the type's lowest value is a number like others."""
    V = 9000
    g = torch.Generator(device=DEV).manual_seed(5)
    rows = torch.randn(7, V, generator=g, device=DEV)
    rows[0, 10:] = -math.inf
    rows[1] = -math.inf
    rows[1, 8000] = 2.0
    rows[2] = -math.inf                                    # nothing left
    rows[3, 4000:] = torch.finfo(torch.float32).min
    rows[4] = torch.finfo(torch.float32).min
    rows[5, 77] = math.inf
    rows[6, ::2] = -math.inf
    tokens = torch.tensor([3, 8000, 5, 4000, 1, 77, 0], dtype=torch.int32, device=DEV)
    got = check(rows, tokens, 20)
    assert got.logprobs[1].item() == 0.0 and got.entropy[1].item() == 0.0
    assert got.logprobs[2].isnan() and got.logprobs[5].isnan() and got.logprobs[6].item() == -math.inf


def test_nan_rows():
    from mini_sglang_b200 import ops
    rows = torch.randn(3, 5000, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    whole = rows[1].clone()
    rows[0, 4321] = math.nan
    rows[2] = math.nan
    rows[2, 17] = 1.0
    got = ops.token_logprobs(rows, torch.zeros(3, dtype=torch.int32, device=DEV), 3)
    assert got.logprobs.isnan().tolist() == [True, False, True] and got.entropy.isnan().tolist() == [True, False, True]
    clean = rows[0].nan_to_num(nan=-math.inf)
    assert got.top_tokens[0].tolist() == clean.topk(3).indices.tolist() and got.top_logprobs[0].isnan().all()
    assert got.top_tokens[1].tolist() == whole.topk(3).indices.tolist()
    assert got.top_tokens[2].tolist() == [17, -1, -1]


def test_tokens_outside_and_large_logits():
    from mini_sglang_b200 import ops
    rows = torch.randn(4, 600, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) * 1e4
    tokens = torch.tensor([-1, 600, 2 ** 31 - 1, 5], dtype=torch.int32, device=DEV)
    got = check(rows, tokens, 2)
    assert got.logprobs.isnan().tolist() == [True, True, True, False]
    assert ops.token_logprobs(rows[:0], tokens[:0], 2).top_tokens.shape == (0, 2)


def test_rows_far_apart():
    """A row offset beyond 32 bits."""
    from mini_sglang_b200 import ops
    big = torch.empty(3 * 800_000_000, dtype=torch.bfloat16, device=DEV)
    rows = big.as_strided((3, 1000), (1_150_000_000, 1))
    rows.copy_(torch.randn(3, 1000, device=DEV))
    check(rows, torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV), 4)
    del big, rows
    torch.cuda.empty_cache()
    assert ops is not None


def test_graph_and_stream():
    """Captured and replayed on other logits, beside the same call on another stream."""
    from mini_sglang_b200 import ops
    a, tok = torch.randn(2, 40000, device=DEV), torch.tensor([5, 6], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    ops.token_logprobs(a, tok, 5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.token_logprobs(a, tok, 5)
    for _ in range(3):
        a.copy_(torch.randn(2, 40000, device=DEV))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = ops.token_logprobs(a, tok, 5)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, beside))
        assert torch.equal(got.top_tokens.long(), plain(a, tok, 5)[3])
