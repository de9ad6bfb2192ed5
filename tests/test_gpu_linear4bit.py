"""``Linear4bit`` (``nsm_linear4bit``) against the definition in 64 bits.

Bound of one output, with A = sum_k |x_k| |w_k| in 64 bits:

* the output's own rounding, ``eps / 2`` of its type relative to the value;
* the fp32 accumulation: at most ``K / 16`` tensor-core adds inside the groups, two
  more per group and one per partial sum (fewer than 64), each off by at most 2^-23 of the
  running magnitude (truncation included), which A bounds;
* the weights: exact for integers, 2^-11 of each value where a codebook is
  rounded to fp16 (fp16 and bf16 outputs), 2^-22 where it is kept as two fp16;
* x: exact for fp16 and bf16, 2^-22 for fp32 (two fp16).
"""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from next_step_ai_b200 import _lib

    _lib.load()
    return torch.device("cuda", 0)


def _make(N, K, gs, kind, dev, seed, scale_dtype=FS, bias=None):
    gen = torch.Generator(device=dev).manual_seed(seed)
    groups = -(-K // gs)
    p = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=dev, generator=gen)
    sc = ((torch.rand((N, groups), device=dev, generator=gen) + 0.5) * 0.02).to(scale_dtype)
    code = zeros = None
    if kind == "code":
        from next_step_ai_b200.nf4 import nf4_code
        code = nf4_code(dev)
    elif kind == "zeros":
        zeros = torch.randint(0, 16, (N, groups), dtype=torch.uint8, device=dev, generator=gen)
    b = torch.randn(N, device=dev, generator=gen).to(bias) if bias is not None else None
    return p, sc, code, zeros, b


def _dense(p, sc, code, zeros, N, K, gs):
    """The weight in 64 bits, from its definition."""
    q = torch.empty((N, K), dtype=torch.int64, device=p.device)
    q[:, 0::2] = (p.reshape(N, K // 2) >> 4).long()
    q[:, 1::2] = (p.reshape(N, K // 2) & 15).long()
    grp = torch.arange(K, device=p.device) // gs
    v = code.double()[q] if code is not None else q.double() - (zeros.double()[:, grp] if zeros is not None else 8.0)
    return v * sc.double()[:, grp]


def _check(y, x, W, bias, code):
    xd = x.double().reshape(-1, x.shape[-1])
    ref = xd @ W.t()
    A = xd.abs() @ W.abs().t()
    if bias is not None:
        ref, A = ref + bias.double(), A + bias.double().abs()
    K = W.shape[1]
    rel = (K / 16 + 2 * K / 32 + 64) * 2.0 ** -23
    if code is not None:
        rel += 2.0 ** -22 if y.dtype == FS else 2.0 ** -11
    if x.dtype == FS:
        rel += 2.0 ** -22
    # a result below the type's smallest normal number is rounded to its subnormal step
    bound = torch.finfo(y.dtype).eps / 2 * (ref.abs() + rel * A) + rel * A + torch.finfo(y.dtype).tiny
    err = (y.double().reshape(ref.shape) - ref).abs()
    worst = float((err / bound).max())
    assert worst <= 1.0, f"error is {worst:.3g} of its bound"
    # and, over all outputs, the error is the rounding of the type (not the worst-case sum)
    typical = {BF: 2.5e-3, FH: 4e-4, FS: 1.5e-6}[y.dtype]
    assert float(err.norm() / ref.norm()) <= typical


CASES = [
    # N, K, group, kind, rows, x, out, scales, bias
    (1, 2, 32, "code", 1, BF, BF, FS, None),
    (1, 2, 32, "sym", 1, FS, FS, FS, FS),
    (16, 128, 128, "sym", 8, FH, FH, FH, None),
    (17, 130, 64, "zeros", 9, BF, BF, BF, BF),
    (255, 1000, 32, "code", 3, FH, FH, FS, FH),
    (257, 1026, 96, "zeros", 5, FS, FS, FH, None),
    (1001, 2086, 128, "zeros", 3, FH, FH, FH, FH),
    (640, 4096, 256, "sym", 17, BF, FS, FS, None),
    (512, 4096, 4096, "sym", 1, BF, BF, FH, BF),
    (333, 640, 1024, "zeros", 2, BF, BF, FH, None),       # one group, wider than the row
    (1024, 16384, 64, "code", 1, BF, BF, FS, None),
    (1024, 16384, 64, "code", 32, BF, BF, FS, None),
    (4096, 4096, 64, "code", 8, BF, FS, FS, None),
    (4096, 1024, 64, "code", 16, FS, FS, FS, FS),         # 32 columns: value + remainder
    (40, 53248, 128, "zeros", 4, BF, BF, BF, None),       # few rows, a long sum
    (5000, 256, 32, "sym", 24, FH, FS, FS, None),
]


@pytest.mark.parametrize("N,K,gs,kind,rows,xd,od,sd,bd", CASES)
def test_matches_definition(dev, N, K, gs, kind, rows, xd, od, sd, bd):
    from next_step_ai_b200.linear4bit import Linear4bit

    p, sc, code, zeros, b = _make(N, K, gs, kind, dev, N + K + rows, sd, bd)
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=gs, code=code, zeros=zeros, bias=b)
    gen = torch.Generator(device=dev).manual_seed(rows)
    x = torch.randn((rows, K), device=dev, generator=gen)
    x[:, ::13] *= 30.0
    x = x.to(xd)
    y = layer(x, out_dtype=od)
    assert y.shape == (rows, N) and y.dtype == od
    W = _dense(p, sc, code, zeros, N, K, gs)
    _check(y, x, W, b, code)
    assert torch.equal(y, layer(x, out_dtype=od))                      # the same bits every time
    alone = torch.cat([layer(x[r:r + 1], out_dtype=od) for r in range(rows)])
    assert torch.equal(y, alone)                                       # rows do not depend on each other


def test_shapes_strides_and_many_rows(dev):
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 300, 514
    p, sc, code, _, _ = _make(N, K, 64, "code", dev, 3)
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code)
    W = _dense(p, sc, code, None, N, K, 64)
    big = torch.randn((70, K + 7), device=dev, dtype=BF)
    y = layer(big[:, 3:3 + K])                     # rows further apart, a base that is aligned to 2 bytes only
    _check(y, big[:, 3:3 + K], W, None, code)      # 70 rows: three passes
    assert torch.equal(y, layer(big[:, 3:3 + K].contiguous()))
    t = torch.randn((K, 5), device=dev, dtype=BF).t()                  # columns are not contiguous
    _check(layer(t), t, W, None, code)
    e = big[:1, :K].expand(4, K)                                       # rows on top of each other
    assert torch.equal(layer(e), layer(e.contiguous()))
    assert layer(big[:, :K].reshape(2, 5, 7, K)).shape == (2, 5, 7, N)
    assert layer(big[0, :K]).shape == (N,)
    assert layer(big[:0, :K]).shape == (0, N)


@pytest.mark.parametrize("xd", [BF, FS])
def test_range_of_x(dev, xd):
    """Values far outside of fp16's range, and rows with infinities and NaN: each
    row has its own scale and touches no other."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 200, 384
    p, sc, _, zeros, _ = _make(N, K, 128, "zeros", dev, 11)
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=128, zeros=zeros)
    W = _dense(p, sc, None, zeros, N, K, 128)
    x = torch.randn((6, K), device=dev)
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3] = 0.0
    x[4, 7] = float("inf")
    x[5, 9] = float("nan")
    x = x.to(xd)
    y = layer(x, out_dtype=FS)
    _check(y[:3], x[:3], W, None, None)
    assert torch.equal(y[3], torch.zeros_like(y[3]))
    hit = W[:, 7] != 0
    assert torch.equal(y[4][hit], torch.sign(W[hit, 7]).float() * float("inf"))
    assert torch.isnan(y[4][~hit]).all() and torch.isnan(y[5]).all()


def test_extreme_zero_points_and_codebooks(dev):
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 64, 256
    p, sc, _, _, _ = _make(N, K, 64, "sym", dev, 5)
    zeros = torch.full((N, 4), 255, dtype=torch.uint8, device=dev)
    zeros[::2] = 0
    x = torch.randn((4, K), device=dev, dtype=BF)
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, zeros=zeros)
    _check(layer(x, out_dtype=FS), x, _dense(p, sc, None, zeros, N, K, 64), None, None)
    for mul in (1e-6, 1e5):                        # a codebook of any magnitude
        code = torch.linspace(-1.0, 0.9, 16, device=dev) * mul
        layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code)
        W = _dense(p, sc, code, None, N, K, 64)
        _check(layer(x, out_dtype=FS), x, W, None, code)
        _check(layer(x), x, W, None, code)


def test_streams_and_graphs(dev):
    """Two streams at once and two graphs captured from one layer, replayed
    together: no scratch memory is shared."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 2048, 4096
    p, sc, code, _, _ = _make(N, K, 64, "code", dev, 8)
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code)
    xs = [torch.randn((r, K), device=dev, dtype=BF) for r in (1, 8)]
    want = [layer(x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(x))
        graphs.append(g)
    for x in xs:
        x.copy_(torch.randn_like(x))
    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_construction(dev, tmp_path):
    from next_step_ai_b200.checkpoint import Nf4Param
    from next_step_ai_b200.linear4bit import Linear4bit
    from next_step_ai_b200.nf4 import dequantize_nf4, nf4_code, quantize_nf4

    N, K = 128, 512
    w = torch.randn((N, K), device=dev) * 0.02
    x = torch.randn((3, K), device=dev, dtype=BF)
    packed, absmax = quantize_nf4(w, nf4_code(dev), 64)
    W = dequantize_nf4(packed, absmax, nf4_code(dev), 64).reshape(N, K).double()
    layer = Linear4bit.from_dense(w)
    _check(layer(x), x, W, None, layer.code)
    param = Nf4Param("w", packed.cpu(), absmax.cpu(), nf4_code(), N, K, 64, "nf4", "bfloat16")
    assert torch.equal(Linear4bit.from_param(param, dev)(x), layer(x))
    whole = Linear4bit.from_dense(w, group_size=128, kind="int4")
    s = w.reshape(N, 4, 128).abs().amax(-1) / 7.0
    Wi = (torch.round(w.reshape(N, 4, 128) / s[..., None]).clamp(-7, 7).double() * s.double()[..., None]).reshape(N, K)
    _check(whole(x), x, Wi, None, None)
    assert whole.weight_bytes() == N * K // 2 + 4 * N * 4


def test_agrees_with_the_lm_head(dev):
    """The same NF4 bytes through the framework's NF4 head: both are within their
    bounds of the product, the head's being the fp16 rounding of the codebook."""
    from next_step_ai_b200.linear4bit import Linear4bit
    from next_step_ai_b200.lm_head import Nf4LmHead

    N, K = 1000, 1024
    p, sc, code, _, _ = _make(N, K, 64, "code", dev, 2)
    x = torch.randn((4, K), device=dev, dtype=BF)
    a = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code)(x, out_dtype=FS)
    b = Nf4LmHead(p, sc, code, out_features=N, in_features=K)(x, out_dtype=FS)
    A = x.double().abs() @ _dense(p, sc, code, None, N, K, 64).abs().t()
    assert bool(((a - b).double().abs() <= 2.0 ** -11 * A + (K / 16 + K / 16 + 128) * 2.0 ** -23 * A).all())


def test_refuses_bad_calls_before_any_launch(dev):
    from next_step_ai_b200 import _lib
    from next_step_ai_b200.linear4bit import Linear4bit

    p, sc, code, zeros, _ = _make(32, 128, 64, "zeros", dev, 1)
    mk = dict(out_features=32, in_features=128, group_size=64)
    layer = Linear4bit(p, sc, zeros=zeros, **mk)
    with pytest.raises(RuntimeError, match="expects 128"):
        layer(torch.zeros((2, 64), device=dev, dtype=BF))
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        layer(torch.zeros((2, 128), device=dev, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        layer(torch.zeros((2, 128), dtype=BF))
    with pytest.raises(RuntimeError, match="no zero points"):
        Linear4bit(p, sc, zeros=zeros, code=torch.zeros(16, device=dev), **mk)
    with pytest.raises(RuntimeError, match="scales has"):
        Linear4bit(p, sc[:, :1], **mk)
    with pytest.raises(RuntimeError, match="bias has"):
        Linear4bit(p, sc, bias=torch.zeros(31, device=dev), **mk)
    lib, x, y = _lib.load(), torch.zeros((33, 128), device=dev, dtype=BF), torch.zeros((33, 32), device=dev, dtype=BF)
    need = lib.nsm_linear4bit_workspace_bytes(32, _lib.NSM_BF16, 32, 128)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)

    def call(rows=2, stride=128, nbytes=need, at=ws.data_ptr(), out_stride=32):
        return lib.nsm_linear4bit(x.data_ptr(), _lib.NSM_BF16, rows, stride, layer._ref, y.data_ptr(), _lib.NSM_BF16,
                                  out_stride, at, nbytes, 0)

    assert need > 0 and lib.nsm_linear4bit_workspace_bytes(33, _lib.NSM_BF16, 32, 128) == 0
    assert call(rows=33) == _lib.NSM_ERR_UNSUPPORTED
    assert call(rows=-1) == _lib.NSM_ERR_INVALID_ARG
    assert call(stride=64) == _lib.NSM_ERR_INVALID_ARG
    assert call(out_stride=31) == _lib.NSM_ERR_INVALID_ARG
    assert call(nbytes=64) == _lib.NSM_ERR_WORKSPACE
    assert call(at=ws.data_ptr() + 16) == _lib.NSM_ERR_WORKSPACE
    assert call(rows=0) == _lib.NSM_OK
    assert call() == _lib.NSM_OK


def test_largest_finite_x(dev):
    """Values next to the top of bf16's and fp32's range, scaled like any other: one and
    many rows (the kernel's own tiles of x, and those of the kernel before it)."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 130, 256
    p, sc, _, zeros, _ = _make(N, K, 128, "zeros", dev, 12)
    sc = sc * 2.0 ** -20
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=128, zeros=zeros)
    W = _dense(p, sc, None, zeros, N, K, 128)
    for xd, rows in ((BF, 1), (BF, 9), (FS, 2), (FS, 16)):
        x = torch.randn((rows, K), device=dev).clamp_(-4, 4)
        x[:, 5] = 4.0
        x = (x * (0.99 * 2.0 ** 126)).to(xd)
        _check(layer(x, out_dtype=FS), x, W, None, None)


@pytest.mark.parametrize("kind,N,K", [("code", 4096, 2048), ("sym", 2048, 16384), ("zeros", 5000, 640)])
def test_a_row_gives_the_same_bits_alone_and_among_others(dev, kind, N, K):
    from next_step_ai_b200.linear4bit import Linear4bit

    p, sc, code, zeros, _ = _make(N, K, 64, kind, dev, 21)
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code, zeros=zeros)
    x = torch.randn((32, K), device=dev, dtype=BF)
    y = layer(x, out_dtype=FS)
    for n in (1, 3, 8, 16, 17):
        assert torch.equal(layer(x[:n], out_dtype=FS), y[:n])


def test_graphs_with_many_rows(dev):
    """Two graphs of one layer whose calls go through the kernel that lays x out, one of them
    in three passes, replayed on two streams at once."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 1030, 2048
    p, sc, _, zeros, b = _make(N, K, 128, "zeros", dev, 31, FH, BF)
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=128, zeros=zeros, bias=b)
    W = _dense(p, sc, None, zeros, N, K, 128)
    xs = [torch.zeros((r, K), device=dev, dtype=t) for r, t in ((9, FS), (70, BF))]
    graphs, outs = [], []
    for x in xs:
        layer(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(x))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in range(3):
        for x in xs:
            x.copy_(torch.randn(x.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed)))
        torch.cuda.synchronize()
        for _ in range(4):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for x, y in zip(xs, outs):
            _check(y, x, W, b, None)


def test_offsets_past_32_bits(dev):
    """A weight of more than 2^32 bytes (its last rows), and rows of x that lie further apart."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 131072 + 133, 65536 + 130
    p = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=dev)
    groups = -(-K // 128)
    sc = (torch.rand((N, groups), device=dev) + 0.5).to(BF)
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=128)
    far = torch.empty(2 ** 31 + K, dtype=BF, device=dev)
    x = torch.as_strided(far, (2, K), (2 ** 31, 1))
    x.copy_(torch.randn((2, K), device=dev))
    y = layer(x, out_dtype=FS)
    for a in (0, 65536, N - 200):
        W = _dense(p[a:a + 200], sc[a:a + 200], None, None, 200, K, 128)
        _check(y[:, a:a + 200], x, W, None, None)


@pytest.mark.parametrize("N,K", [(512, 128), (513, 2048), (2048, 2050), (4096, 4096), (4100, 4096), (9216, 1024),
                                 (37888, 256), (38000, 256), (75776, 128), (75777, 128)])
def test_weights_in_one_launch_and_in_two(dev, N, K):
    """The sizes at which a row block goes from a cluster of 16 CTAs to fewer, and to partials: one,
    eight, nine and 32 rows, and fp32 rows in two columns each."""
    from next_step_ai_b200.linear4bit import Linear4bit

    for kind in ("code", "zeros"):
        p, sc, code, zeros, b = _make(N, K, 64, kind, dev, N + K, FS, FS)
        layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code, zeros=zeros, bias=b)
        W = _dense(p, sc, code, zeros, N, K, 64)
        for rows, xd in ((1, BF), (8, FH), (9, BF), (32, BF), (4, FS), (16, FS)):
            x = torch.randn((rows, K), device=dev).to(xd)
            y = layer(x, out_dtype=FS)
            _check(y, x, W, b, code)
            assert torch.equal(y, layer(x, out_dtype=FS))


def _infinite_check(y, x, W):
    """Infinite, and of that sign, where the definition is; NaN where that is; else finite."""
    ref = x.double() @ W.t()
    assert torch.equal(torch.isnan(y), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(torch.isinf(y), inf) and torch.equal(y[inf].double(), ref[inf])


@pytest.mark.parametrize("rows", [1, 12])
@pytest.mark.parametrize("xd,od", [(BF, FS), (FS, FS), (BF, BF), (FH, FH), (FS, FH)])
def test_infinite_x_with_a_codebook(dev, rows, xd, od):
    """One infinity in a row: an infinity of the weight's sign, or NaN where the weight is 0."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 300, 384
    p, sc, code, _, _ = _make(N, K, 64, "code", dev, 41)
    code = code.clone()
    code[2] = 2.0 ** -33                               # next to nothing, but not nothing
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code)
    W = _dense(p, sc, code, None, N, K, 64)
    for value in (float("inf"), -float("inf")):
        x = torch.randn((rows, K), device=dev).to(xd)
        x[0, 77] = value
        x[-1, 200] = value
        x[rows // 2, 77] = value
        _infinite_check(layer(x, out_dtype=od), x, W)


@pytest.mark.parametrize("rows", [1, 12])
@pytest.mark.parametrize("xd,od", [(BF, FS), (FS, FS), (BF, BF), (FS, BF)])
def test_infinite_codebook_entries(dev, rows, xd, od):
    """An infinite entry gives infinities where a weight uses it, and touches nothing else."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 48, 128
    p, sc, code, _, _ = _make(N, K, 64, "code", dev, 9)
    code = code.clone()
    code[15] = float("inf")
    q = _dense(p, torch.ones_like(sc), torch.arange(16.0, device=dev), None, N, K, 64)
    p = torch.where((q[:, 0::2] == 15) | (q[:, 1::2] == 15), 0, p.reshape(N, K // 2)).contiguous()
    p[3, 7] = 0xF1
    W = _dense(p, sc, code, None, N, K, 64)
    x = (torch.rand((rows, K), device=dev) + 0.5).to(xd)
    x[0, 14] *= -1.0
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code)
    _infinite_check(layer(x, out_dtype=od), x, W)
    x[-1, 14] = float("inf")
    _infinite_check(layer(x, out_dtype=od), x, W)


def _one_column_rows(dev, rows, K, dtype):
    """Rows with a single 1.0 each, in different columns."""
    x = torch.zeros((rows, K), device=dev, dtype=dtype)
    at = (torch.arange(rows, device=dev) * 37 + 5) % K
    x[torch.arange(rows, device=dev), at] = 1.0
    return x, at


@pytest.mark.parametrize("N,K,rows", [(700, 320, 1), (700, 320, 12), (4096, 4096, 8), (1024, 8192, 32)])
@pytest.mark.parametrize("xd,od", [(BF, BF), (FH, FH), (BF, FH), (FS, FS)])
def test_one_column_gives_the_weight_rounded_once(dev, N, K, rows, xd, od):
    """A row of x with a single 1.0 gives a column of W: off by the output's rounding, 2^-22 for
    the codebook as two fp16, and 2^-23 for the product with the scale (at most 2^-24 each of
    two roundings); the other columns add exact zeros."""
    from next_step_ai_b200.linear4bit import Linear4bit

    p, sc, code, _, _ = _make(N, K, 64, "code", dev, N + rows)
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code)
    W = _dense(p, sc, code, None, N, K, 64)
    x, at = _one_column_rows(dev, rows, K, xd)
    ref = W[:, at].t()
    rel = 2.0 ** -22 + 2.0 ** -23
    bound = (torch.finfo(od).eps / 2 * (1 + rel) + rel) * ref.abs()
    assert bool(((layer(x, out_dtype=od).double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("od", [BF, FH, FS])
def test_codebook_rounded_to_fp16_where_asked(dev, od):
    """``fp16_code``: the definition with a codebook that fp16 rounded, in any output type; a power
    of two before the rounding keeps it out of the subnormal numbers."""
    from next_step_ai_b200.linear4bit import Linear4bit

    for N, K, rows in ((700, 322, 1), (4096, 4096, 8), (1030, 2048, 32)):
        p, sc, code, _, b = _make(N, K, 64, "code", dev, N + rows, FS, FS)
        mk = dict(out_features=N, in_features=K, group_size=64, code=code, bias=b)
        layer = Linear4bit(p, sc, fp16_code=True, **mk)
        x = torch.randn((rows, K), device=dev, dtype=BF)
        y = layer(x, out_dtype=od)
        _check(y, x, _dense(p, sc, (code * 64).half().float() / 64, None, N, K, 64), b, code)
        if od == FS:
            assert not torch.equal(y, Linear4bit(p, sc, **mk)(x, out_dtype=od))
        x[0, 9] = float("inf")
        _infinite_check(layer(x, out_dtype=od)[:1], x[:1], _dense(p, sc, code, None, N, K, 64))
    with pytest.raises(RuntimeError, match="with a codebook"):
        Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, fp16_code=True)
    w = torch.randn((64, 128), device=dev)
    a, c = Linear4bit.from_dense(w, fp16_code=True), Linear4bit.from_dense(w)
    x = torch.randn((2, 128), device=dev)
    assert not torch.equal(a(x), c(x))


@pytest.mark.parametrize("xd", [BF, FS])
@pytest.mark.parametrize("kind,mul", [("code", 1.0), ("code", 1.7e-3), ("sym", 1.0)])
def test_tiny_x(dev, xd, kind, mul):
    """Rows down to 1e-35: as exact as others (a result is at least 2^-120 or so, a normal number),
    whether the kernel lays x out itself (one row, eight) or not.  The two give the same bits where
    results are 2^-100 and more.  Below, sums on the way may be subnormal numbers in the first
    (those of an fp32 x's remainders, 2^-11 of the others and less, before the rest): they round by
    up to 2^-150, and that can turn a later rounding, of a sum of any size, by a whole step of its
    own.  Both stay within the definition's bound."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 300, 512
    p, sc, code, _, _ = _make(N, K, 64, kind, dev, 51)
    code = code * mul if code is not None else None
    sc = sc / mul
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code)
    W = _dense(p, sc, code, None, N, K, 64)
    many = 16 if xd == FS else 32
    for size in (1e-27, 1e-30, 1e-32, 1e-33, 1e-34, 1e-35):
        x = (torch.randn((many, K), device=dev) * size).to(xd)
        y = layer(x, out_dtype=FS)
        # (the definition's bound times 2^60: _check allows a smallest normal number otherwise)
        _check(y.double().mul(2.0 ** 60).float(), x.float() * 2.0 ** 60, W, None, code)
        for n in (1, 3, many // 4):
            own, same = layer(x[:n], out_dtype=FS), y[:n].abs() >= 2.0 ** -100
            assert size < 1e-27 or bool(same.any())
            assert torch.equal(own[same], y[:n][same])
            _check(own.double().mul(2.0 ** 60).float(), x[:n].float() * 2.0 ** 60, W, None, code)


def test_large_x_with_small_scales(dev):
    """Products of x and the codebook past fp32's range, brought back by the scales."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 130, 256
    p, sc, code, _, _ = _make(N, K, 64, "code", dev, 52)
    code, sc = code * 2.0 ** 20, sc * 2.0 ** -40
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code)
    W = _dense(p, sc, code, None, N, K, 64)
    for xd, rows in ((BF, 1), (BF, 9), (FS, 2), (FS, 16)):
        x = (torch.randn((rows, K), device=dev) * 2.0 ** 120).to(xd)
        _check(layer(x, out_dtype=FS), x, W, None, code)


@pytest.mark.parametrize("kind", ["code", "zeros"])
def test_arguments_may_be_overwritten(dev, kind):
    """The layer holds copies of all that it was made from, in calls and in a captured graph."""
    from next_step_ai_b200.linear4bit import Linear4bit

    N, K = 300, 256
    made = _make(N, K, 64, kind, dev, 61, FS, FS)
    p, sc, code, zeros, b = made
    layer = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, code=code, zeros=zeros, bias=b)
    x = torch.randn((3, K), device=dev, dtype=BF)
    want = layer(x, out_dtype=FS)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(x, out_dtype=FS)
    for t in made:
        if t is not None:
            t.fill_(3)
    assert torch.equal(layer(x, out_dtype=FS), want)
    g.replay()
    assert torch.equal(y, want)
    strided = torch.randn((N, 2), device=dev)
    a = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, bias=strided[:, 0])
    c = Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, bias=strided[:, 0].contiguous())
    assert torch.equal(a(x), c(x)) and a.bias.is_contiguous()
