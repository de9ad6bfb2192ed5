"""``nsm_linear4bit`` when its waits run out: without a GPU fault, every wait gives up at
once (``nsm_linear4bit_set_wait_limit(-1)``).  Copies that were asked for are waited for
with the ordinary limit before a CTA ends, and the next call is as if nothing had been."""
from __future__ import annotations

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


@pytest.fixture
def no_tries(dev):
    """Sets the limit to none; the ordinary one is back after the test."""
    from next_step_ai_b200 import _lib

    lib = _lib.load()

    def set_to(tries):
        torch.cuda.synchronize()
        _lib.check(lib.nsm_linear4bit_set_wait_limit(tries), "nsm_linear4bit_set_wait_limit")

    yield set_to
    set_to(0)


def _layer(dev, N, K, kind, fp16_code=False):
    from next_step_ai_b200.linear4bit import Linear4bit
    from next_step_ai_b200.nf4 import nf4_code

    gen = torch.Generator(device=dev).manual_seed(N + K)
    p = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=dev, generator=gen)
    sc = (torch.rand((N, -(-K // 64)), device=dev, generator=gen) + 0.5) * 0.02
    z = torch.randint(0, 16, sc.shape, dtype=torch.uint8, device=dev, generator=gen) if kind == "zeros" else None
    return Linear4bit(p, sc, out_features=N, in_features=K, group_size=64, zeros=z, fp16_code=fp16_code,
                      code=nf4_code(dev) if kind == "code" else None)


# a cluster's CTAs and partials; the kernel's own tiles of x and those laid out before; rings of
# three and four places; fewer units than places, and many
@pytest.mark.parametrize("N,K", [(40, 128), (600, 2048), (4096, 4096), (4096, 16384), (20000, 1024)])
@pytest.mark.parametrize("kind,fp16_code", [("code", False), ("code", True), ("zeros", False), ("sym", False)])
@pytest.mark.parametrize("rows,xd", [(1, BF), (8, FH), (9, BF), (16, FS)])
def test_waits_that_give_up_at_once(dev, no_tries, N, K, kind, fp16_code, rows, xd):
    layer = _layer(dev, N, K, kind, fp16_code)
    x = torch.randn((rows, K), device=dev).to(xd)
    want = layer(x)
    no_tries(-1)
    y = layer(x)
    no_tries(0)
    assert bool(torch.isnan(y).all())
    assert torch.equal(layer(x), want)


@pytest.mark.parametrize("N,K,rows,xd", [(4096, 4096, 1, BF), (4096, 4096, 9, BF), (4096, 16384, 1, FS),
                                         (4096, 16384, 16, FS)])
@pytest.mark.parametrize("kind", ["code", "zeros"])
def test_a_failed_wait_is_recorded(dev, no_tries, N, K, rows, xd, kind):
    """The word keeps the failure over later calls, of any layer on the device, and until it is read."""
    from next_step_ai_b200 import _lib

    layer, other = _layer(dev, N, K, kind), _layer(dev, 40, 128, kind)
    x = torch.randn((rows, K), device=dev).to(xd)
    layer.error()
    layer(x)
    assert layer.error() == 0
    no_tries(-1)
    layer(x)
    no_tries(0)
    layer(x)
    assert other.error() == _lib.NSM_ERR_TIMEOUT
    assert other.error() == 0 and layer.error() == 0


def test_a_search_tells_of_its_heads_failure(dev, no_tries):
    """A failed head's NaN logits are no candidates: the search says so, and a head without an error
    word has none."""
    from next_step_ai_b200 import BeamSearch, _lib

    head = _layer(dev, 1000, 256, "code")
    search = BeamSearch(head, 2, 3, max_tokens=8)
    head.error()
    hidden = torch.randn((6, 256), device=dev, dtype=BF)
    search.step(hidden)
    assert search.error() == 0
    no_tries(-1)
    search.step(hidden)
    no_tries(0)
    search.step(hidden)
    assert search.error() == _lib.NSM_ERR_TIMEOUT and search.error() == 0

    class Plain:
        device = dev

        def __call__(self, hidden, out_dtype):
            return torch.zeros((hidden.shape[0], 50), device=dev, dtype=out_dtype)

    assert BeamSearch(Plain(), 2, 3, max_tokens=8).error() == 0


@pytest.mark.parametrize("tries", [1, 2, 8])
@pytest.mark.parametrize("N,K,rows,xd", [(4096, 4096, 1, BF), (4096, 16384, 1, BF), (4096, 16384, 8, FH),
                                         (4096, 16384, 9, BF), (20000, 2048, 16, FS), (700, 16384, 32, BF)])
@pytest.mark.parametrize("kind", ["code", "zeros"])
def test_few_tries(dev, no_tries, tries, N, K, rows, xd, kind):
    """Waits that may run out in the middle of a run, or not: an output is right or NaN, and where any
    is NaN the failure is recorded."""
    from next_step_ai_b200 import _lib

    layer = _layer(dev, N, K, kind)
    x = torch.randn((rows, K), device=dev).to(xd)
    want = layer(x)
    layer.error()
    no_tries(tries)
    got = [layer(x) for _ in range(10)]
    no_tries(0)
    code = layer.error()
    lost = [torch.isnan(y) for y in got]
    assert all(torch.equal(torch.where(m, want, y), want) for m, y in zip(lost, got))
    assert code == (_lib.NSM_ERR_TIMEOUT if any(bool(m.any()) for m in lost) else code)
    assert torch.equal(layer(x), want) and layer.error() == 0
