"""``ops.sample`` against a restatement in 64 bits, and its refusals.

The restatement sorts each row, applies the filters one after another on
float64 weights and walks the running sums.  Tokens must be equal: both sides
hold the weights to about 2^-45 of the largest, so a token could only differ if
a uniform fell within about 1e-11 of a border, and the uniforms here are
seeded.  The log-probability is a float32 sum of V exponentials and one log:
its error is at most a few float32 rounding steps of the sum (each thread adds
at most V / 512 + 16 terms in a row, 2^-24 of the running sum each, plus expf's
2 ulp) and one of the result: 1e-5 absolute + 2^-22 relative covers V = 131,072.
"""

import math

import numpy as np
import pytest
import torch

from sheetsage2_refined_b200 import ops

gpu = pytest.mark.gpu


def draw64(x, allowed, u, t, k, p, m):
    """(token, logprob) of one row in float64; ``x`` float32 values (bias added)."""

    index = np.nonzero(allowed)[0]
    x = x[index].astype(np.float64)
    if x.size and np.isnan(x).any():
        return int(index[np.isnan(x)][0]), math.nan
    if not x.size or x.max() == -math.inf:
        return 0, -math.inf
    best = x.max()
    if best == math.inf:
        return int(index[x == math.inf][0]), 0.0
    logz = math.log(np.exp(x - best).sum())
    if not t > 0:
        return int(index[np.argmax(x)]), -logz
    w = np.exp((x - best) / t)
    order = np.argsort(-x, kind="stable")
    sw = w[order].copy()
    if k > 0:
        sw[k:] = 0
    if p < 1:
        cum = np.cumsum(sw)
        keep = cum - sw < max(p, 0.0) * cum[-1]
        keep[0] = True
        sw[~keep] = 0
    if m > 0:
        sw[sw < min(m, 1.0)] = 0
    kept = np.zeros_like(w)
    kept[order] = sw
    run = np.cumsum(kept)
    u = u if u > 0 else 0.0
    hit = np.nonzero(run > u * run[-1])[0]
    i = int(hit[0]) if hit.size else int(np.nonzero(kept)[0][-1])
    return int(index[i]), x[i] - best - logz


def expect(logits, uniforms, bias, allowed, t, k, p, m):
    rows, vocab = logits.shape
    x = logits.float()
    if bias is not None:
        x = x + bias
    x = x.numpy()
    ok = np.ones((rows, vocab), bool) if allowed is None else np.broadcast_to(allowed.numpy() != 0, (rows, vocab))

    def at(v, r):
        return float(v[r]) if isinstance(v, torch.Tensor) else float(np.float32(v))

    got = [draw64(x[r], ok[r], float(uniforms[r]), at(t, r), int(at(k, r)), at(p, r), at(m, r)) for r in range(rows)]
    return torch.tensor([g[0] for g in got]), torch.tensor([g[1] for g in got], dtype=torch.float64)


def check(logits, uniforms, bias=None, allowed=None, t=1.0, k=0, p=1.0, m=0.0):
    want, logp = expect(logits, uniforms, bias, allowed, t, k, p, m)

    def cuda(v):
        return v.cuda() if isinstance(v, torch.Tensor) else v

    tokens, lp = ops.sample(logits.cuda(), uniforms.cuda(), temperature=cuda(t), top_k=cuda(k), top_p=cuda(p),
                            min_p=cuda(m), bias=cuda(bias), allowed=cuda(allowed))
    tokens, lp = tokens.cpu(), lp.cpu().double()
    assert torch.equal(tokens, want), [(r, int(tokens[r]), int(want[r])) for r in
                                       torch.nonzero(tokens != want)[:8, 0].tolist()]
    both = torch.isfinite(logp)
    assert torch.equal(torch.isnan(lp), torch.isnan(logp))
    assert torch.equal(lp[~both & ~torch.isnan(lp)], logp[~both & ~torch.isnan(lp)])
    assert bool(((lp - logp)[both].abs() <= 1e-5 + 2.0**-22 * logp[both].abs()).all()), (lp - logp)[both].abs().max()


def inputs(rows, vocab, dtype, seed, masked=True):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, vocab, generator=g) * 2 + 9.0 * (torch.rand(rows, vocab, generator=g) < 10 / vocab))
    allowed = torch.rand(rows, vocab, generator=g) < 0.4 if masked else None
    bias = torch.randn(vocab, generator=g).round() if masked else None
    return logits.to(dtype), torch.rand(rows, generator=g), bias, allowed


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 100, 0.8, 0.02),
           (0.0, 5, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (2.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 10**9, 0.999, 0.0)]


@gpu
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (2, 513), (17, 2048), (6, 4097), (3, 32576), (300, 700)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_draws_match_the_definition(rows, vocab, dtype):
    for i, (t, k, p, m) in enumerate(FILTERS):
        logits, u, bias, allowed = inputs(rows, vocab, dtype, 100 * vocab + i, masked=i % 2 == 0)
        check(logits, u, bias, allowed, t, k, p, m)


@gpu
@pytest.mark.parametrize("rows,vocab", [(1, 32576), (150, 9000), (300, 32576), (3, 131071)])
@pytest.mark.parametrize("t,k,p,m", [(1.0, 700, 1.0, 0.0), (1.5, 1500, 0.9, 0.0), (2.0, 5000, 1.0, 0.001), (3.0, 8999, 0.99, 0.0),
                                     (5.0, 0, 0.97, 0.0), (0.01, 300, 0.9, 0.0), (1e9, 0, 0.5, 0.0), (1e-30, 40, 0.5, 0.1)])
def test_filters_that_keep_many_tokens_and_extreme_temperatures(rows, vocab, t, k, p, m):
    """Past the lists' sizes: the searches over the whole row take over."""

    for masked in (False, True):
        logits, u, bias, allowed = inputs(rows, vocab, torch.float32, k + vocab, masked=masked)
        if masked:  # whole spans, as a grammar's classes: some CTAs' shares hold nothing
            span = torch.arange(vocab) * 9 // vocab
            allowed = allowed & (torch.rand(rows, 9, generator=torch.Generator().manual_seed(k)) < 0.4)[:, span]
        check(logits, u, bias, allowed, t, k, p, m)
    coarse, u, _, _ = inputs(rows, vocab, torch.float32, k, masked=False)
    check(torch.round(coarse), u, None, None, t, k, p, m)  # a dozen values: thousands of ties at any threshold


@gpu
@pytest.mark.parametrize("vocab", [131071, 524288])
def test_large_vocabularies(vocab):
    for i, (t, k, p, m) in enumerate(FILTERS[:5]):
        logits, u, bias, allowed = inputs(2, vocab, torch.bfloat16, i, masked=i % 2 == 1)
        check(logits, u, bias, allowed, t, k, p, m)


@gpu
def test_per_row_parameters_and_rows_beyond_range():
    rows = 64
    logits, u, bias, allowed = inputs(rows, 5000, torch.float32, 7)
    g = torch.Generator().manual_seed(8)
    t = torch.rand(rows, generator=g) * 2
    k = torch.randint(0, 300, (rows,), generator=g, dtype=torch.int32)
    p = torch.rand(rows, generator=g) * 1.2
    m = torch.rand(rows, generator=g) * 0.2
    t[0], t[1] = 0.0, 1e-3
    check(logits, u, bias, allowed, t, k, p, m)
    # out of range: as the documented nearest value
    t[2], k[3], p[4], p[5], m[6], m[7] = -1.0, -5, 3.0, -1.0, -0.5, 2.0
    u[8], u[9], u[10], u[11] = 0.0, 1.0, -3.0, 5.0
    u[8] = u[10] = 0.0  # a negative uniform counts as 0
    want = [x.clone() for x in (u, p, m, k)]
    check(logits, u, bias, allowed, t, k, p, m)
    u[10] = -3.0
    tokens, _ = ops.sample(logits.cuda(), u.cuda(), temperature=t.cuda(), top_k=k.cuda(), top_p=p.cuda(),
                           min_p=m.cuda(), bias=bias.cuda(), allowed=allowed.cuda())
    expected, _ = expect(logits, want[0], bias, allowed, t, k, p, m)
    assert torch.equal(tokens.cpu(), expected)


@gpu
@pytest.mark.parametrize("t,k,p,m", FILTERS)
def test_ties_empty_rows_and_special_values(t, k, p, m):
    vocab = 6000
    g = torch.Generator().manual_seed(3)
    logits = torch.round(torch.randn(16, vocab, generator=g) * 2) / 2
    allowed = torch.rand(16, vocab, generator=g) < 0.5
    allowed[0] = False
    logits[1] = -math.inf
    logits[2, [40, 4000]] = math.nan
    allowed[2, [40, 4000]] = True
    logits[3, [77, 5999]] = math.inf
    allowed[3, [77, 5999]] = True
    logits[4] = 0.0  # every token ties
    logits[5, ::2], logits[5, 1::2] = 0.0, -0.0
    logits[6] = torch.finfo(torch.float32).min  # the type's lowest value, a live token all the same
    logits[7, :] = -math.inf
    logits[7, 3000] = -5.0
    allowed[7, 3000] = True
    logits[8, ~allowed[8]] = math.nan  # masked places hold NaN and infinities
    logits[9, ~allowed[9]] = math.inf
    allowed[10] = False
    allowed[10, vocab - 1] = True
    logits[11] = torch.finfo(torch.float32).max
    logits[12, 17] = torch.finfo(torch.float32).max
    allowed[12, 17] = True
    u = torch.rand(16, generator=g)
    check(logits, u, None, allowed, t, k, p, m)


@gpu
def test_strided_rows_broadcast_mask_and_given_outputs():
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(9, 4100, generator=g)
    u = torch.rand(9, generator=g)
    mask = torch.rand(3001, generator=g) < 0.5
    view = wide[:, 7:3008]
    want, _ = expect(view, u, None, mask[None], 0.9, 30, 0.95, 0.0)
    dev = wide.cuda()
    out = torch.full((12,), -7, dtype=torch.int64, device="cuda")
    lp = torch.full((12,), 3.0, device="cuda")
    tokens, _ = ops.sample(dev[:, 7:3008], u.cuda(), temperature=0.9, top_k=30, top_p=0.95, allowed=mask.cuda(),
                           out=out[:9], logprobs=lp[:9])
    assert tokens.data_ptr() == out.data_ptr()
    assert torch.equal(out[:9].cpu(), want)
    assert out[9:].tolist() == [-7] * 3 and lp[9:].tolist() == [3.0] * 3  # rows behind the last are left alone
    one = dev[:1, :2000].expand(5, -1)  # the same logits for every row (stride 0)
    u5 = torch.linspace(0, 0.99, 5)
    want, _ = expect(one.cpu().contiguous(), u5, None, None, 1.0, 0, 1.0, 0.0)
    assert torch.equal(ops.sample(one, u5.cuda())[0].cpu(), want)


@gpu
def test_frequencies_follow_the_weights():
    """65,536 uniforms on an even grid: the counts are the weights to one grid step each (no chance involved)."""

    x = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5])
    n = 65536
    u = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    tokens, _ = ops.sample(x.cuda()[None].expand(n, -1), u.float().cuda(), temperature=0.8)
    w = torch.softmax(x.double() / 0.8, 0)
    counts = torch.bincount(tokens.cpu(), minlength=5).double()
    assert bool(((counts - w * n).abs() <= 2.0).all()), counts - w * n


@gpu
def test_streams_overlapping_calls_and_graph_replay():
    logits, u, bias, allowed = inputs(33, 9000, torch.float32, 11)
    args = dict(temperature=0.9, top_k=70, top_p=0.9, bias=bias.cuda(), allowed=allowed.cuda())
    x, uu = logits.cuda(), u.cuda()
    want, want_lp = ops.sample(x, uu, **args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(ops.sample(x, uu, **args))
    torch.cuda.synchronize()
    for tokens, lp in got:
        assert torch.equal(tokens, want) and torch.equal(lp, want_lp)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, lp = ops.sample(x, uu, **args)
    uu.copy_(1 - uu)
    graph.replay()
    torch.cuda.synchronize()
    again, _ = expect(logits, uu.cpu(), bias, allowed, 0.9, 70, 0.9, 0.0)
    assert torch.equal(tokens.cpu(), again)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_nans_of_either_sign_and_masked_ones(dtype):
    x = torch.zeros(5, 700, dtype=dtype)
    ints = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    wide = {torch.float32: 0xFFC00001 - 2**32, torch.bfloat16: 0xFFC1 - 2**16, torch.float16: 0xFE01 - 2**16}[dtype]
    ints[0, 300] = wide  # a negative NaN with a payload
    ints[1, 300], x[1, 650] = wide, math.nan
    x[2, 12], ints[2, 600] = math.nan, wide
    ints[3, 300] = wide
    x[4], x[4, ::3] = -0.0, 0.0
    allowed = torch.ones(5, 700, dtype=torch.bool)
    allowed[3, 300] = False
    tokens, lp = ops.sample(x.cuda(), torch.full((5,), 0.5, device="cuda"), allowed=allowed.cuda())
    # rows 3 and 4: equal weights, the middle one of 699 and of 700 tokens
    assert tokens.tolist() == [300, 300, 12, 350, 350]
    assert lp[:3].isnan().all() and (lp[3:].cpu() + torch.tensor([699.0, 700.0]).log()).abs().max() < 1e-5
