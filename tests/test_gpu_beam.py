"""``beam_select``, ``BeamStates`` and ``BeamSearch`` against their definitions.

Scores: |error| <= eps/2 of fp32 relative to the score (the output's rounding), plus
the error of the logsumexp: the sum of exponentials is off by at most 2^-21 (the
hardware's exponential and its argument's rounding) plus 2^-24 for each of the additions one
thread and the block's tree make, relative to the sum, which is the absolute error of its
logarithm.  Tokens and parents are compared for equality; two candidates whose scores
in 64 bits differ by less than that bound may swap, which the test accepts only then."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32
INF = math.inf


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from next_step_ai_b200 import _lib

    _lib.load()
    return torch.device("cuda", 0)


def _totals(logits, scores, finished, pad):
    """[B, W * V] in 64 bits, -infinity where there is no candidate."""
    B, W = scores.shape
    d = logits.double().reshape(B, W, -1)
    d = torch.where(torch.isnan(d), -INF, d).clamp(max=float(torch.finfo(FS).max))
    m = d.amax(-1, keepdim=True)
    m = torch.where(m == -INF, 0.0, m)
    lse = m + torch.log(torch.exp(d - m).sum(-1, keepdim=True))
    s = scores.double()[..., None]
    t = torch.where((d == -INF) | ~(s > -INF), -INF, s + (d - lse))
    if finished is not None:
        t = torch.where(finished[..., None], -INF, t)
        t[..., pad] = torch.where(finished & (scores > -INF), scores.double(), t[..., pad])
    return t.reshape(B, -1)


def _check(got, logits, scores, k, finished=None, pad=0, exact=False):
    gs, gt, gp = got
    B, W = scores.shape
    V = logits.shape[-1]
    assert gs.shape == gt.shape == gp.shape == (B, k)
    assert gs.dtype == FS and gt.dtype == gp.dtype == torch.int64
    tot = _totals(logits, scores, finished, pad)
    ref, at = torch.sort(tot, dim=-1, descending=True, stable=True)
    pad_cols = max(0, k - ref.shape[1])
    ref = torch.nn.functional.pad(ref, (0, pad_cols), value=-INF)[:, :k]
    at = torch.nn.functional.pad(at, (0, pad_cols))[:, :k]
    gone = ref == -INF
    assert torch.equal(gs == -INF, gone)
    assert bool((gt[gone] == -1).all()) and bool((gp[gone] == 0).all())
    live = ~gone
    bound = 2.0 ** -21 + (16 * (V // 8192 + 1) + 64) * 2.0 ** -24
    err = (gs.double() - ref).abs()[live]
    fin = torch.isfinite(ref[live])
    assert bool((err[fin] <= 2.0 ** -24 * ref[live][fin].abs() + bound).all())
    assert not bool(fin.any()) or float(err[fin].max()) <= 2.0 ** -24 * float(ref[live][fin].abs().max()) + 2e-6
    flat = (gp * V + gt)
    if exact:
        assert torch.equal(flat[live], at[live])
        return
    same = flat == at
    mine = torch.gather(tot, 1, torch.where(gone, 0, flat))
    assert bool((same | gone | ((mine - ref).abs() <= 2 * bound)).all())
    for b in range(B):                                  # every candidate once
        f = flat[b][live[b]]
        assert f.unique().numel() == f.numel()
    assert float((same | gone).float().mean()) > 0.999


def _inputs(B, W, V, dtype, dev, seed, tail=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn((B, W, V + tail), device=dev, generator=gen) * 3.0).to(dtype)
    s = -10.0 * torch.rand((B, W), device=dev, generator=gen)
    return x[..., :V], s, gen


@pytest.mark.parametrize("B,W,V,k,dtype,tail", [
    (1, 1, 1, 1, FS, 0), (1, 1, 7, 16, BF, 0), (2, 3, 31, 64, FH, 5), (1, 4, 128256, 8, FS, 0), (3, 5, 50257, 10, FH, 0),
    (2, 5, 50257, 10, BF, 47), (16, 8, 32000, 16, BF, 0), (1, 32, 8191, 64, FS, 0), (2, 32, 8193, 33, BF, 7),
    (40, 16, 1000, 17, FH, 0), (300, 2, 16384, 4, BF, 0), (1, 1, 400001, 64, FS, 3), (4, 4, 24576, 1, FS, 0)])
def test_matches_definition(dev, B, W, V, k, dtype, tail):
    from next_step_ai_b200 import beam_select

    x, s, gen = _inputs(B, W, V, dtype, dev, B * 7 + W + V, tail)
    got = beam_select(x, s, num_candidates=k)
    _check(got, x, s, k)
    again = beam_select(x, s, num_candidates=k)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    # some beams finished, some out
    f = torch.rand((B, W), device=dev, generator=gen) < 0.3
    s2 = torch.where(torch.rand((B, W), device=dev, generator=gen) < 0.3, -INF, s)
    pad = V // 2
    _check(beam_select(x, s2, num_candidates=k, finished=f, pad_token=pad), x, s2, k, f, pad)


def test_equal_values_go_by_index(dev):
    """Nothing but ties: one value in all of the vocabulary and all beams (every
    list overflows), a few values, and beams that are the same."""
    from next_step_ai_b200 import beam_select

    for B, W, V, k in ((1, 1, 100000, 64), (2, 32, 20000, 64), (1, 3, 128256, 5)):
        x = torch.full((B, W, V), 1.5, device=dev, dtype=BF)
        s = torch.zeros((B, W), device=dev)
        _check(beam_select(x, s, num_candidates=k), x, s, k, exact=True)
        g = torch.Generator(device=dev).manual_seed(V)
        x = torch.randint(0, 3, (B, 1, V), device=dev, generator=g).to(FH).expand(B, W, V)  # the same row for each beam
        _check(beam_select(x, s, num_candidates=k), x, s, k, exact=True)
        x = x.contiguous()[..., 1:]                                                          # and unaligned
        _check(beam_select(x, s, num_candidates=k), x, s, k, exact=True)
    x = torch.tensor([[[0.0, -0.0, -1.0, 0.0]]], device=dev)                                 # -0 equals 0
    assert beam_select(x, torch.zeros((1, 1), device=dev), num_candidates=3)[1].tolist() == [[0, 1, 3]]


@pytest.mark.parametrize("order", ["up", "down", "late"])
def test_sorted_logits(dev, order):
    """The best at the end of the row: each tile replaces the list."""
    from next_step_ai_b200 import beam_select

    V = 100003
    v = torch.arange(V, device=dev, dtype=FS) * 1e-3
    x = v if order == "up" else v.flip(0) if order == "down" else torch.where(v > 99.0, v, -v)
    x = x.reshape(1, 1, V).repeat(2, 2, 1)
    x[:, 1] -= 0.25
    s = torch.tensor([[0.0, -1e-4], [-3.0, -2.0]], device=dev)
    for k in (1, 16, 40, 64):
        _check(beam_select(x, s, num_candidates=k), x, s, k)


def test_masked_infinite_and_nan_logits(dev):
    from next_step_ai_b200 import beam_select

    B, W, V = 2, 6, 30011
    x, s, gen = _inputs(B, W, V, FS, dev, 1)
    x[0, 0] = -INF                                       # nothing may come
    x[0, 1, :] = -INF
    x[0, 1, 29000:29003] = torch.tensor([1.0, 2.0, 2.0], device=dev)
    x[0, 2, ::3] = float("nan")
    x[0, 3, 12345] = INF
    x[0, 3, 20000] = INF
    x[0, 4] = float("nan")
    x[0, 5, 100] = torch.finfo(FS).min                   # a mask of the lowest value is a candidate
    x[1, :, 8192:] = torch.finfo(FS).min
    x[1, 0, :] = torch.finfo(FS).min
    for k in (4, 12, 64):
        _check(beam_select(x, s, num_candidates=k), x, s, k)
    got = beam_select(x[:1], torch.tensor([[-INF, -1.0, -INF, -INF, 0.0, float("nan")]], device=dev), num_candidates=8)
    assert got[1].tolist() == [[29001, 29002, 29000, -1, -1, -1, -1, -1]]
    assert got[2].tolist() == [[1, 1, 1, 0, 0, 0, 0, 0]]
    # rows that are out or finished are not read: NaN in them does no harm
    f = torch.tensor([[True] * 5 + [False], [False] * 6], device=dev)
    _check(beam_select(x, s, num_candidates=10, finished=f, pad_token=9), x, s, 10, f, 9)
    big = torch.tensor([[[1e5, 1e5 - 2.0, -1e5, 3.3e38, 3.3e38]]], device=dev)
    _check(beam_select(big, torch.zeros((1, 1), device=dev), num_candidates=5), big, torch.zeros((1, 1), device=dev), 5)


def test_views_streams_and_graphs(dev):
    from next_step_ai_b200 import beam_select

    B, W, V = 4, 4, 40000
    x, s, gen = _inputs(B, W, V, BF, dev, 9)
    want = beam_select(x, s)
    assert want[0].shape == (B, 2 * W)
    assert all(torch.equal(a, b) for a, b in zip(beam_select(x.reshape(B * W, V), s), want))
    t = x.transpose(0, 1).contiguous().transpose(0, 1)   # beams outermost in memory
    assert all(torch.equal(a, b) for a, b in zip(beam_select(t, s), want))
    c = x.transpose(1, 2).contiguous().transpose(1, 2)   # the vocabulary is not contiguous
    assert all(torch.equal(a, b) for a, b in zip(beam_select(c, s), want))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    y = torch.randn_like(x)
    want_y = beam_select(y, s)
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(beam_select(x if i == 0 else y, s))
    torch.cuda.synchronize()
    for i, w in enumerate((want, want_y)):
        assert all(torch.equal(a, b) for g in got[i] for a, b in zip(g, w))
    graphs, outs, ins = [], [], [x.clone(), y.clone()]
    for q in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(beam_select(q, s))
        graphs.append(g)
    ins[0].copy_(y)
    ins[1].copy_(x)
    torch.cuda.synchronize()
    for g, st in zip(graphs, streams):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, (want_y, want)):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
    none = beam_select(x[:0], s[:0])
    assert none[1].shape == (0, 2 * W)


def test_select_refusals(dev):
    from next_step_ai_b200 import beam_select

    x, s = torch.zeros((2, 3, 10), device=dev), torch.zeros((2, 3), device=dev)
    for bad, text in ((dict(num_candidates=0), "candidates"), (dict(num_candidates=65), "candidates"),
                      (dict(pad_token=10), "pad_token"), (dict(pad_token=-1), "pad_token"),
                      (dict(finished=torch.zeros((2, 2), device=dev, dtype=torch.bool)), "finished"),
                      (dict(finished=torch.zeros((2, 3), device=dev)), "finished")):
        with pytest.raises(RuntimeError, match=text):
            beam_select(x, s, **bad)
    with pytest.raises(RuntimeError, match="scores must be"):
        beam_select(x, s.double())
    with pytest.raises(RuntimeError, match="logits has shape"):
        beam_select(x[:, :2], s)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        beam_select(x.double(), s)
    with pytest.raises(RuntimeError, match="1 to 32 beams"):
        beam_select(torch.zeros((1, 33, 4), device=dev), torch.zeros((1, 33), device=dev))


def _moved(t, parents, length_dim=None, length=None):
    """The definition, on a copy."""
    B, W = parents.shape
    out = t.clone()
    for b in range(B):
        for w in range(W):
            src = int(parents[b, w])
            if not 0 <= src < W:
                continue
            d, f = out[b * W + w], t[b * W + src]
            if length_dim is not None and length is not None:
                d, f = d.narrow(length_dim - 1, 0, length), f.narrow(length_dim - 1, 0, length)
            d.copy_(f)
    return out


def _state(shape, dtype, dev, gen):
    return torch.randint(-100, 100, shape, device=dev, generator=gen).to(dtype)


@pytest.mark.parametrize("B,W", [(1, 1), (1, 2), (3, 4), (2, 7), (1, 16), (2, 17), (1, 32)])
def test_reorder(dev, B, W):
    """Every element size and alignment, strided states, lengths from none to all."""
    from next_step_ai_b200 import BeamStates

    gen = torch.Generator(device=dev).manual_seed(B * 100 + W)
    R = B * W
    wide = _state((R, 3, 20, 24), BF, dev, gen)
    odd = _state((R, 77), torch.uint8, dev, gen)
    seq = _state((9, R, 6), FS, dev, gen)
    states = [
        (_state((R, 2, 33, 40), BF, dev, gen), 2),              # a cache [rows, heads, positions, dim]
        (wide[:, :, 2:19, 8:16], None),                         # two strided dimensions
        (wide.clone()[:, 1], 1),                                # one head of a wider cache
        (_state((R, 33), torch.int64, dev, gen), 1),            # a history
        (odd[:, 1:], None),                                     # bytes at odd addresses
        (_state((R, 3, 5, 35), FH, dev, gen), 3),               # positions last, 2 bytes each
        (seq.transpose(0, 1), None),                            # rows in the middle of memory
        (_state((R,), torch.bool, dev, gen), None),
        (_state((R, 4099), FS, dev, gen), None),
        (_state((R, 64, 3), torch.float64, dev, gen), 1),
    ]
    ts, dims = [t for t, _ in states], [d for _, d in states]
    handle = BeamStates(ts, B, W, dims)
    assert handle.max_length == 20
    for length in (None, 20, 13, 1, 0):
        parents = torch.randint(0, W, (B, W), device=dev, generator=gen)
        if length == 13:
            parents = torch.arange(W, device=dev).flip(0).repeat(B, 1)       # a cycle: nobody stays
        if length == 1 and W > 1:
            parents[0, 0], parents[-1, -1] = -1, W                           # no such beams
        whole = [wide.clone(), odd.clone(), seq.clone()]
        want = [_moved(t, parents, d, length) for t, d in zip(ts, dims)]
        handle.reorder_(parents, length)
        torch.cuda.synchronize()
        for i, (t, w) in enumerate(zip(ts, want)):
            assert torch.equal(t, w), (i, length)
        # what is around a view stays as it was
        whole[0][:, :, 2:19, 8:16] = wide[:, :, 2:19, 8:16]
        whole[1][:, 1:] = odd[:, 1:]
        assert torch.equal(whole[0], wide) and torch.equal(whole[1], odd)


def test_reorder_large_offsets_and_graph(dev):
    """A state of over 4 GB (offsets pass 32 bits), and a captured reorder."""
    from next_step_ai_b200 import BeamStates

    B, W = 2, 4
    big = torch.empty((B * W, 600_000_000), dtype=torch.uint8, device=dev)
    for r in range(B * W):
        big[r] = r + 1
    handle = BeamStates([big], B, W)
    parents = torch.tensor([[0, 0, 3, 2], [3, 1, 1, 0]], device=dev)
    handle.reorder_(parents)
    want = [1, 1, 4, 3, 8, 6, 6, 5]
    for r in range(B * W):
        assert int(big[r].min()) == int(big[r].max()) == want[r]
    del big, handle
    t = torch.arange(B * W * 1000, device=dev).reshape(B * W, 1000)
    handle = BeamStates([t], B, W, [1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        handle.reorder_(parents, 600)
    before = t.clone()
    parents.copy_(torch.tensor([[1, 2, 3, 0], [0, 1, 2, 2]], device=dev))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(t, _moved(before, parents, 1, 600))


def test_reorder_refusals(dev):
    from next_step_ai_b200 import BeamStates

    t = torch.zeros((6, 4, 8), device=dev)
    h = BeamStates([t], 2, 3, [1])
    p = torch.zeros((2, 3), dtype=torch.int64, device=dev)
    with pytest.raises(RuntimeError, match="parents must be"):
        h.reorder_(p.int())
    with pytest.raises(RuntimeError, match="parents must be"):
        h.reorder_(p[:1])
    for n in (-1, 5):
        with pytest.raises(RuntimeError, match="outside"):
            h.reorder_(p, n)
    with pytest.raises(RuntimeError, match="outside"):
        BeamStates([t], 2, 3).reorder_(p, 2)


def test_search_steps_match_a_plain_search(dev):
    """Head, selection and reordering together, with a caller's cache: every step
    equals a plain beam search on the same logits, states included."""
    from next_step_ai_b200 import BeamSearch, Linear4bit

    B, W, H, V, steps, eos = 3, 4, 128, 500, 12, 7
    gen = torch.Generator(device=dev).manual_seed(4)
    head = Linear4bit.from_dense(torch.randn((V, H), device=dev, generator=gen) * 0.3)
    embed = torch.randn((V, H), device=dev, generator=gen).to(BF)
    cache = torch.zeros((B * W, 2, steps, 16), device=dev, dtype=BF)
    search = BeamSearch(head, B, W, max_tokens=steps, eos_token=eos, pad_token=eos, states=[cache], length_dims=[2])
    scores = torch.full((B, W), -INF, device=dev)
    scores[:, 0] = 0
    finished = torch.zeros((B, W), dtype=torch.bool, device=dev)
    hist = torch.zeros((B * W, 0), dtype=torch.int64, device=dev)
    mirror = cache.clone()
    hidden = torch.randn((B, 1, H), device=dev, generator=gen).to(BF).expand(B, W, H).reshape(B * W, H).contiguous()
    for i in range(steps):
        cache[:, :, i] = hidden[:, :32].reshape(B * W, 2, 16)
        mirror[:, :, i] = hidden[:, :32].reshape(B * W, 2, 16)
        logits = head(hidden, out_dtype=FS)
        tokens = search.step(hidden, i + 1)
        ref, at = torch.sort(_totals(logits, scores, finished, eos), dim=-1, descending=True, stable=True)
        par, tok = at[:, :W] // V, at[:, :W] % V
        assert torch.equal(tokens, tok)
        scores = search.scores.clone()
        assert torch.allclose(scores.double(), ref[:, :W], atol=2e-5)
        rows = (par + W * torch.arange(B, device=dev)[:, None]).reshape(-1)
        hist = torch.cat([hist[rows], tok.reshape(-1, 1)], dim=1)
        mirror = mirror[rows]
        finished = torch.gather(finished, 1, par) | (tok == eos)
        assert torch.equal(search.finished, finished)
        assert torch.equal(cache[:, :, :i + 1], mirror[:, :, :i + 1])
        assert torch.equal(search.sequences().reshape(B * W, -1), hist)
        hidden = (hidden[rows] * 0.5 + embed[tok.reshape(-1)]).to(BF)
    with pytest.raises(RuntimeError, match="history holds"):
        search.step(hidden)
    search.reset()
    assert search.length == 0 and search.sequences().shape == (B, W, 0)


def test_search_over_the_sparse_mlp_and_nf4_head(dev):
    """The framework's own path with beams as rows: router, union MLP, NF4 head,
    selection.  Beams of one prompt start equal, so step one is one beam's."""
    from next_step_ai_b200 import BeamSearch, RouterWeights, SparseMlpWeights, route_sparse_mlp, union_decode
    from next_step_ai_b200.lm_head import Nf4LmHead
    from next_step_ai_b200.nf4 import nf4_code, quantize_nf4

    B, W, H, I, V = 2, 4, 512, 1024, 1000
    gen = torch.Generator(device=dev).manual_seed(2)
    code = nf4_code(dev)

    def q(n, k):
        return quantize_nf4(torch.randn((n, k), device=dev, generator=gen) * 0.05, code, 64)

    (gp, ga), (up, ua), (dp, da) = q(I, H), q(I, H), q(H, I)
    weights = SparseMlpWeights.from_bnb_rowmajor(hidden=H, intermediate=I, gate_packed=gp, gate_absmax=ga, up_packed=up,
                                                 up_absmax=ua, down_packed=dp, down_absmax=da, code=code.cpu(),
                                                 tiled=True)
    nb = I // 32
    router = RouterWeights(enc_w=torch.randn((64, H), device=dev, generator=gen).to(BF) * 0.05,
                           enc_b=None, score_w=torch.randn((nb, 64), device=dev, generator=gen).to(BF),
                           score_b=None, top_k=8, basis_top_k=64)
    hp, ha = q(V, H)
    head = Nf4LmHead(hp, ha, code, out_features=V, in_features=H)
    embed = torch.randn((V, H), device=dev, generator=gen).to(BF)
    search = BeamSearch(head, B, W, max_tokens=4)
    hidden = torch.randn((B, 1, H), device=dev, generator=gen).to(BF).expand(B, W, H).reshape(B * W, H).contiguous()
    scores = None
    for i in range(4):
        y = union_decode(hidden, route_sparse_mlp(hidden, router), weights)
        hidden = (hidden + y.to(BF)).contiguous()
        tokens = search.step(hidden)
        assert tokens.shape == (B, W) and int(tokens.min()) >= 0 and int(tokens.max()) < V
        if i == 0:
            lp = torch.log_softmax(head(hidden[::W], out_dtype=FS).double(), -1)
            top = torch.topk(lp, W, dim=-1)
            assert torch.equal(tokens, top.indices)
            assert torch.allclose(search.scores.double(), top.values, atol=1e-5)
        else:
            assert bool((search.scores.max(1).values <= scores.max(1).values).all())
        scores = search.scores.clone()
        hidden = embed[tokens.reshape(-1)]
    assert search.sequences().shape == (B, W, 4)


@pytest.mark.parametrize("W,V,k", [(1, 800, 32), (1, 1024, 64), (16, 900, 32), (3, 1500, 64), (32, 500, 64)])
def test_small_vocabularies(dev, W, V, k):
    """Fewer blocks of the vocabulary than candidates, with spread and with few values."""
    from next_step_ai_b200 import beam_select

    x, s, gen = _inputs(3, W, V, FS, dev, V + k)
    _check(beam_select(x, s, num_candidates=k), x, s, k)
    x = torch.randint(0, 4, (3, W, V), device=dev, generator=gen).to(FH)
    s = torch.zeros((3, W), device=dev)
    same = x[:, :1].expand(3, W, V)
    _check(beam_select(same, s, num_candidates=k), same, s, k, exact=True)


@pytest.mark.parametrize("B", [1, 7, 8, 15, 16, 33, 34, 74, 75, 148, 149])
def test_batches_in_one_launch_and_in_two(dev, B):
    """The sizes at which a selection goes from clusters of 16 CTAs per item to fewer, and to
    two launches: what an item gets does not depend on its neighbours but for rounding."""
    from next_step_ai_b200 import beam_select

    x, s, gen = _inputs(B, 3, 5003, FH, dev, B)
    _check(beam_select(x, s, num_candidates=6), x, s, 6)
    x[:] = x[:1, :1].clone()                           # every beam alike: ties by beam, then token
    s = torch.zeros_like(s)
    _check(beam_select(x, s, num_candidates=6), x, s, 6, exact=True)


def test_logits_shared_far_apart_and_other_layouts(dev):
    """Beams that share their logits (stride 0), rows more than 2^31 values apart, scores and
    flags that are views, bytes as flags."""
    from next_step_ai_b200 import beam_select

    x, s, gen = _inputs(2, 4, 3001, BF, dev, 77)
    shared = x[:, :1].expand(2, 4, 3001)
    _check(beam_select(shared, s, num_candidates=9), shared, s, 9)
    far = torch.empty(2 ** 31 + 16384, dtype=BF, device=dev)
    view = torch.as_strided(far, (2, 4, 3001), (2 ** 31, 3001, 1))
    view.copy_(x)
    f = torch.rand((2, 4), device=dev, generator=gen) < 0.4
    want = beam_select(x.contiguous(), s, num_candidates=9, finished=f, pad_token=5)
    wide = torch.zeros((4, 2, 2), device=dev)
    wide[..., 0] = s.t()
    flags = f.t().contiguous().t().to(torch.uint8) * 7
    got = beam_select(view, wide[..., 0].t(), num_candidates=9, finished=flags, pad_token=5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    _check(got, x, s, 9, f, 5)


@pytest.mark.parametrize("B,W,V,k,dtype", [(28, 11, 1429, 15, BF), (8, 16, 1712, 29, BF), (21, 7, 1370, 12, FS),
                                           (1, 5, 3041, 10, FH), (160, 5, 3296, 9, FS), (2, 3, 40000, 64, FH)])
def test_few_blocks_with_many_values_above_the_last(dev, B, W, V, k, dtype):
    """As many blocks of the vocabulary as candidates, some of them far below the others: the
    last one's largest value says little about the candidates."""
    from next_step_ai_b200 import beam_select

    x, s, gen = _inputs(B, W, V, dtype, dev, V + k)
    _check(beam_select(x, s * 20, num_candidates=k), x, s * 20, k)
    down = torch.sort(x.float(), dim=-1, descending=True).values.to(dtype)
    _check(beam_select(down, s, num_candidates=k), down, s, k)
    f = torch.rand((B, W), device=dev, generator=gen) < 0.4
    _check(beam_select(down, s, num_candidates=k, finished=f, pad_token=3), down, s, k, f, 3)


def test_states_that_share_memory(dev):
    """Parts of one buffer are put in order as states of their own; parts that share bytes are refused."""
    from next_step_ai_b200 import BeamStates

    B, W = 2, 3
    kv = torch.randn((B * W, 2, 4, 8, 6), device=dev)
    want = kv.clone()
    parents = torch.tensor([[1, 1, 0], [2, 0, 2]], device=dev)
    rows = (parents + W * torch.arange(B, device=dev)[:, None]).reshape(-1)
    BeamStates([kv[:, 1], kv[:, 0]], B, W, [2, 2]).reorder_(parents, length=5)
    want[:, :, :, :5] = want[rows][:, :, :, :5]
    assert torch.equal(kv, want)
    with pytest.raises(RuntimeError, match="share memory"):
        BeamStates([kv, kv[:, 1]], B, W)
    with pytest.raises(RuntimeError, match="share memory"):
        BeamStates([kv[:, 0], kv[:, :, 2:]], B, W)


@pytest.mark.parametrize("B,W,V,k,dtype", [(1, 4, 128256, 8, FS), (2, 8, 50257, 16, BF), (1, 32, 20000, 64, FS),
                                           (3, 3, 1500, 64, FH), (1, 1, 400001, 64, FS), (9, 5, 4099, 10, BF)])
@pytest.mark.parametrize("words", [0, 1, 3])
def test_words_masked_by_the_lowest_value(dev, B, W, V, k, dtype, words):
    """Fewer words are left than candidates are wanted: the rest are masked words, which the type's
    lowest finite value makes candidates of equal scores, by beam, then token.  With the same scores
    for two beams, and one that is out."""
    from next_step_ai_b200 import beam_select

    gen = torch.Generator(device=dev).manual_seed(V + k)
    x = torch.full((B, W, V), torch.finfo(dtype).min, device=dev, dtype=dtype)
    at = torch.randint(0, V, (words,), device=dev, generator=gen)
    x[..., at] = torch.randn((B, W, words), device=dev, generator=gen).to(dtype)
    s = -10.0 * torch.rand((B, W), device=dev, generator=gen)
    s[:, W // 2] = s[:, 0]
    if W > 2:
        s[0, 1] = -INF
    f = torch.zeros((B, W), dtype=torch.bool, device=dev)
    f[-1, -1] = True
    for finished in (None, f):
        got = beam_select(x, s, num_candidates=k, finished=finished, pad_token=V - 1)
        tot = _totals(x, s, finished, V - 1)
        ref, flat = torch.sort(tot, dim=-1, descending=True, stable=True)
        ref, flat = ref[:, :k], flat[:, :k]
        # with at most a few words the sums of exponentials are those of 64 bits to 2^-21; the scores of
        # masked words are near -3e38 (or -65504) and all sums are far below one step of them in fp32:
        # in 64 bits they are equal for beams with equal scores, and else in an order that the sums'
        # errors may change only for finite masks of fp16
        live = ref > -INF
        assert torch.equal(got[0] > -INF, live)
        if dtype != FH:
            assert torch.equal((got[2] * V + got[1])[live], flat[live])
        else:
            mine = torch.gather(tot, 1, (got[2] * V + got[1]).clamp(min=0))
            assert bool((((mine - ref).abs() <= 2.0 ** -18) | ~live).all())


@pytest.mark.parametrize("B,W,V,k,dtype", [(1, 4, 128256, 8, FS), (16, 8, 128256, 16, BF), (1, 32, 128256, 64, FS)])
def test_ties_take_no_longer_than_a_few_passes(dev, B, W, V, k, dtype):
    """A vocabulary of equal values, or masked by the lowest one, against ordinary logits: a few more
    passes over the chosen blocks (measured 2.5 to 6 times; a search bit by bit took 70 to 370)."""
    from next_step_ai_b200 import beam_select

    gen = torch.Generator(device=dev).manual_seed(3)
    s = -torch.rand((B, W), device=dev, generator=gen)
    masked = torch.full((B, W, V), torch.finfo(dtype).min, device=dev, dtype=dtype)
    masked[..., 5] = 1.0
    took = []
    for x in (torch.randn((B, W, V), device=dev, generator=gen).to(dtype), masked, torch.zeros_like(masked)):
        beam_select(x, s, num_candidates=k)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(10):
                beam_select(x, s, num_candidates=k)
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            g.replay()
            a.record()
            g.replay()
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        took.append(best)
    assert max(took[1:]) <= 12 * took[0], took
