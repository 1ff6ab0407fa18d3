"""``ops.shared_attention`` against the formula in float64, and its refusals.

Tolerances.  With P = sum_j p_j |v_j| per output channel (the softmax weights
p sum to 1): the weights are rounded once to the tensors' type (half a step,
eps / 2 relative), the output once more (eps / 2 of its value); the float32
sums run over at most a few thousand terms a chain (2^-12 relative); a score is
a float32 sum of ``dim`` products, off by at most ``ds = dim * 2^-24 * scale *
sum |q k|``, which moves every weight by up to 2 ds.  Hence
|out - exact| <= (eps / 2 + 2^-12 + 2 ds) P + eps / 2 |exact|, and
|lse - exact| <= ds + 2^-14 + 2^-22 |exact|.
"""

import math

import pytest
import torch

from sheetsage2_refined_b200 import ops

gpu = pytest.mark.gpu
PAGE = 64
BF16, F16 = torch.bfloat16, torch.float16


def exact(q, sk, sv, own_k, own_v, table, n, scale):
    """(out, lse, P, ds) in float64, row by row; ``sk``/``sv`` the live shared tokens, tensors on any device."""

    rows, heads, dim = q.shape
    kvh = sk.shape[1]
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64, device=q.device)
    ds = torch.zeros_like(lse)
    group = heads // kvh
    for r in range(rows):
        k, v = sk.double(), sv.double()
        live = max(0, int(n[r])) if n is not None else 0
        if live:
            pages = table[r, : -(-live // PAGE)].long()
            k = torch.cat([k, own_k[pages].double().transpose(1, 2).reshape(-1, kvh, dim)[:live]])
            v = torch.cat([v, own_v[pages].double().transpose(1, 2).reshape(-1, kvh, dim)[:live]])
        if not k.shape[0]:
            continue
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        s = torch.einsum("hd,shd->hs", q[r].double(), k) * scale
        lse[r] = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[r][:, None])
        out[r] = torch.einsum("hs,shd->hd", p, v)
        mass[r] = torch.einsum("hs,shd->hd", p, v.abs())
        ds[r] = torch.einsum("hd,shd->hs", q[r].double().abs(), k.abs()).amax(-1) * (scale * dim * 2.0**-24)
    return out, lse, mass, ds


def assert_close(out, lse, want, dtype):
    o, e, mass, ds = want
    half = torch.finfo(dtype).eps / 2
    tol = (half + 2.0**-12 + 2 * ds[..., None]) * mass + half * o.abs() + 1e-30
    worst = ((out.double() - o).abs() / tol).max().item()
    assert torch.isfinite(out).all() and worst <= 1, worst
    assert torch.equal(torch.isinf(lse), torch.isinf(e))
    f = torch.isfinite(e)
    far = ((lse.double() - e)[f].abs() / (ds + 2.0**-14 + 2.0**-22 * e.abs())[f])
    assert far.numel() == 0 or far.max() <= 1, far.max()


def make(rows, heads, kvh, dim, shared, lens, dtype, seed=0, head_major=True, junk=True):
    """Inputs on the GPU; K/V behind every length is NaN."""

    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    q = (rand(rows, heads, dim) * 1.5).to(dtype)
    kv = []
    for _ in range(2):
        t = (rand(kvh, shared, dim) + rand(kvh, 1, dim)).to(dtype)
        kv.append(t.transpose(0, 1) if head_major else t.transpose(0, 1).contiguous())
    own = {}
    if lens is not None:
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        pages = max(1, -(-max(lens) // PAGE))
        total = rows * pages + 3
        table = torch.randperm(total, generator=g, device="cuda")[: rows * pages].int().view(rows, pages)
        pools = [rand(total, kvh, PAGE, dim).to(dtype) for _ in range(2)]
        if junk:
            keep = torch.zeros(total, PAGE, dtype=torch.bool, device="cuda")
            for r, live in enumerate(lens):
                for p in range(pages):
                    keep[table[r, p], : max(0, min(PAGE, live - p * PAGE))] = True
            for pool in pools:
                pool[~keep[:, None, :, None].expand_as(pool)] = math.nan
            # table entries past a row's pages are garbage
            used = (torch.arange(pages, device="cuda")[None] * PAGE) < n[:, None]
            table = torch.where(used, table, torch.full_like(table, -(2**30)))
        own = dict(own_k=pools[0], own_v=pools[1], page_table=table, own_len=n)
    return q, kv[0], kv[1], own


def check(q, sk, sv, own, dtype, scale=None, **kw):
    out, lse = ops.shared_attention(q, sk, sv, **own, scale=scale, **kw)
    want = exact(q, sk, sv, own.get("own_k"), own.get("own_v"), own.get("page_table"), own.get("own_len"),
                 q.shape[-1] ** -0.5 if scale is None else scale)
    assert_close(out, lse, want, dtype)
    return out, lse


@gpu
@pytest.mark.parametrize("shared", [1, 2, 63, 64, 65, 127, 128, 129, 500, 1499])
@pytest.mark.parametrize("rows", [1, 5, 128, 131])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16)])
def test_shared_only(shared, rows, dim, dtype):
    q, k, v, own = make(rows, 2, 2, dim, shared, None, dtype, seed=shared * 7 + rows)
    check(q, k, v, own, dtype)


@gpu
@pytest.mark.parametrize("heads,kvh", [(1, 1), (6, 2), (8, 1), (5, 5), (20, 2), (16, 1), (24, 3), (40, 1)])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("shared", [0, 70, 300])
def test_grouped_heads_and_own_pages(heads, kvh, dim, dtype, shared):
    lens = [0, 1, 63, 64, 65, 128, 200, 321, 7]
    q, k, v, own = make(len(lens), heads, kvh, dim, shared, lens, dtype, seed=heads + shared, head_major=shared == 70)
    out, lse = check(q, k, v, own, dtype)
    if shared == 0:  # the row without a key
        assert not out[0].any() and bool((lse[0] == -math.inf).all())


@gpu
@pytest.mark.parametrize("rows,lens_max", [(1, 5000), (40, 700), (200, 130)])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16)])
def test_longer_rows(rows, lens_max, dim, dtype):
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, lens_max + 1, (rows,), generator=g).tolist()
    lens[0] = lens_max
    q, k, v, own = make(rows, 4, 2, dim, 777, lens, dtype, seed=rows)
    check(q, k, v, own, dtype)


@gpu
@pytest.mark.parametrize("rows,shared,heads,kvh", [(3, 16384, 2, 2), (300, 4000, 2, 1), (1025, 600, 1, 1)])
def test_long_shared_parts_and_many_rows(rows, shared, heads, kvh):
    for dim, dtype in ((64, BF16), (128, BF16), (64, F16)):
        q, k, v, own = make(rows, heads, kvh, dim, shared, None, dtype, seed=rows)
        check(q, k, v, own, dtype)


@gpu
def test_no_key_anywhere():
    q = torch.randn(4, 3, 64, device="cuda").bfloat16()
    empty = torch.empty(0, 3, 64, dtype=BF16, device="cuda")
    out, lse = ops.shared_attention(q, empty, empty)
    assert not out.any() and bool((lse == -math.inf).all())
    q, k, v, own = make(4, 3, 3, 64, 0, [0, 0, 0, 0], BF16)
    out, lse = ops.shared_attention(q, k, v, **own)
    assert not out.any() and bool((lse == -math.inf).all())


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("live", [-3, 0, 1, 64, 100, 129, 300, 5000])
def test_device_length_of_the_shared_part_hides_what_lies_behind(live, dim):
    q, k, v, own = make(7, 4, 2, dim, 300, [0, 3, 64, 100, 0, 65, 2], BF16, seed=live)
    n = max(0, min(live, 300))
    k, v = k.clone(), v.clone()
    k[n:], v[n:] = math.nan, math.inf
    length = torch.tensor([live], dtype=torch.int32, device="cuda")
    out, lse = ops.shared_attention(q, k, v, **own, shared_len=length)
    want = exact(q, k[:n], v[:n], *(own[x] for x in ("own_k", "own_v", "page_table", "own_len")), dim**-0.5)
    assert_close(out, lse, want, BF16)


@gpu
def test_strides_outputs_and_rows_behind_the_last():
    g = torch.Generator(device="cuda").manual_seed(5)
    big = torch.randn(9, 7, 3, 72, generator=g, device="cuda").half()
    q = big[:, 2, :, 3:67]  # rows and heads apart, not 16-byte aligned
    kv = torch.randn(90, 2, 3, 80, generator=g, device="cuda").half()
    k, v = kv[:, 0, :, 8:72], kv[:, 1, :, 16:80]
    room = torch.full((11, 5, 3, 66), 7.0, device="cuda").half()
    lse = torch.full((12, 3), 7.0, device="cuda")
    out = room[:9, 1, :, 1:65]
    got, _ = ops.shared_attention(q, k, v, out=out, lse=lse[:9])
    assert got.data_ptr() == out.data_ptr()
    want = exact(q, k, v, None, None, None, None, 64**-0.5)
    assert_close(out, lse[:9], want, F16)
    assert bool((room[9:] == 7).all()) and bool((room[:, 0] == 7).all()) and bool((room[..., 65:] == 7).all())
    assert bool((room[..., 0] == 7).all()) and bool((lse[9:] == 7).all())


@gpu
def test_large_scores_and_other_scales():
    """Scores in the hundreds: the running maximum has to move, in either direction of the keys."""

    for order in (1, -1):
        q, k, v, own = make(70, 2, 2, 64, 900, [500] * 70, BF16, seed=3)
        ramp = torch.linspace(0.1, 6, 900, device="cuda")[:, None, None] * order + (0 if order > 0 else 6.1)
        k = (k.float() * ramp).bfloat16()
        check(q, k, v, own, BF16, scale=0.7)
        check(q, k, v, own, BF16, scale=1e-3)


@gpu
@pytest.mark.parametrize("what", ["page", "negative", "length"])
def test_broken_pages_are_reported_and_not_read(what):
    lens = [64, 130, 200, 0]
    q, k, v, own = make(4, 2, 1, 64, 65, lens, BF16, seed=9)
    if what == "length":
        own["own_len"] = own["own_len"].clone()
        own["own_len"][2] = 64 * own["page_table"].shape[1] + 1
    else:
        own["page_table"] = own["page_table"].clone()
        own["page_table"][2, 1] = own["own_k"].shape[0] if what == "page" else -1
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = ops.shared_attention(q, k, v, **own, error=error)
    assert int(error) == (12 if what == "length" else 11)
    assert bool(torch.isnan(out[2]).all()) and bool(torch.isnan(lse[2]).all())
    keep = [0, 1, 3]
    want = exact(q[keep], k, v, own["own_k"], own["own_v"], own["page_table"][keep], own["own_len"][keep], 0.125)
    assert_close(out[keep], lse[keep], want, BF16)


@gpu
def test_offsets_beyond_32_bits():
    """A pool of more than 2^31 elements, the rows' pages at its end."""

    pages = 2**31 // (PAGE * 64) + 8
    pool = torch.zeros(pages, 1, PAGE, 64, dtype=BF16, device="cuda")
    pool[-8:] = torch.randn(8, 1, PAGE, 64, device="cuda").bfloat16()
    table = torch.arange(pages - 8, pages, dtype=torch.int32, device="cuda").view(4, 2)
    n = torch.tensor([100, 128, 1, 65], dtype=torch.int32, device="cuda")
    q = torch.randn(4, 2, 64, device="cuda").bfloat16()
    k = torch.empty_strided((70, 1, 64), (2**25, 64, 1), dtype=BF16, device="cuda").normal_()  # tokens 2^25 apart
    check(q, k, k, dict(own_k=pool, own_v=pool, page_table=table, own_len=n), BF16)


@gpu
def test_calls_are_deterministic_overlap_and_replay():
    q, k, v, own = make(33, 8, 2, 128, 1000, [(37 * r) % 300 for r in range(33)], BF16, seed=2)
    want, want_lse = ops.shared_attention(q, k, v, **own)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(ops.shared_attention(q, k, v, **own))
    torch.cuda.synchronize()
    for o, l in got:
        assert torch.equal(o, want) and torch.equal(l, want_lse)
    length = torch.tensor([1000], dtype=torch.int32, device="cuda")
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.shared_attention(q, k, v, **own, shared_len=length))
        graphs.append(graph)
    for live in (1000, 70, 1000):
        length.fill_(live)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        graphs[0].replay()
        with torch.cuda.stream(side):  # the two graphs at the same time, each on a workspace of its own
            graphs[1].replay()
        torch.cuda.synchronize()
        again, _ = ops.shared_attention(q, k, v, **own, shared_len=length)
        assert torch.equal(outs[0][0], again) and torch.equal(outs[1][0], again)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_k_and_v_in_different_layouts_and_out_in_place(dim):
    """K as [heads, tokens, dim] and V as [tokens, heads, dim] or the other way round; out may be q itself."""

    for k_major in (True, False):
        q, k, v, own = make(20, 6, 3, dim, 333, [(41 * r) % 190 for r in range(20)], F16, seed=12)
        if k_major:
            v = v.contiguous()
        else:
            k = k.contiguous()
        for pages in (own, {}):
            want = exact(q, k, v, *[pages.get(x) for x in ("own_k", "own_v", "page_table", "own_len")], dim**-0.5)
            mine = q.clone()
            out, lse = ops.shared_attention(mine, k, v, **pages, out=mine)
            assert_close(out, lse, want, F16)


@gpu
def test_the_most_rows_and_heads_of_a_call():
    """2^24 (row, head) pairs over one kv head: 131,072 query tiles."""

    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(32768, 512, 64, generator=g, device="cuda", dtype=BF16)
    k, v = (torch.randn(70, 1, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    out, lse = ops.shared_attention(q, k, v)
    for rows in ([0, 1], [16383, 16384], [32766, 32767]):
        assert_close(out[rows], lse[rows], exact(q[rows], k, v, None, None, None, None, 0.125), BF16)


@gpu
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
def test_broadcast_queries_one_page_table_for_all_and_repeated_pages(dim, dtype):
    q, k, v, own = make(6, 4, 2, dim, 200, [256] * 6, dtype, seed=21, junk=False)
    table = own["page_table"][0].clone()
    table[2] = table[0]  # the same page twice in a row
    own["page_table"] = table.expand(6, -1)
    own["own_len"] = torch.tensor([256, 200, 64, 1, 0, 129], dtype=torch.int32, device="cuda")
    check(q[:1].expand(6, -1, -1), k, v, own, dtype)
    check(q[:, :1].expand(-1, 4, -1), k, v, own, dtype)


@gpu
@pytest.mark.parametrize("dim,heads,kvh", [(64, 16, 16), (128, 32, 8)])
def test_short_and_long_shared_parts_beside_own_pages(dim, heads, kvh):
    """Either side of the size up to which the shared part leaves the own part room on the SMs."""

    for shared in (1111, 20000 if dim == 64 else 24000):
        q, k, v, own = make(24, heads, kvh, dim, shared, [(97 * r) % 500 for r in range(24)], BF16, seed=22)
        check(q, k, v, own, BF16)


@gpu
@pytest.mark.parametrize("live", [None, 16000, 5000, 40])
def test_parts_of_unequal_length(live):
    """Few query tiles over a long shared part: the last part of each is shorter, for every live length."""

    q, k, v, _ = make(1000, 16, 16, 64, 16001, None, BF16, seed=23)
    length = None if live is None else torch.tensor([live], dtype=torch.int32, device="cuda")
    out, lse = ops.shared_attention(q, k, v, shared_len=length)
    rows = [0, 127, 128, 511, 999]
    seen = 16001 if live is None else live
    assert_close(out[rows], lse[rows], exact(q[rows], k[:seen], v[:seen], None, None, None, None, 0.125), BF16)
