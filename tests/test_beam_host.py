"""Host side of beam selection and reordering (no GPU): the description of a
state's runs, size queries and refusals."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
from next_step_ai_b200 import _lib, beam  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from next_step_ai_b200.build import build

        build()
    return _lib.load()


def _elements(c, rows, es, length=None):
    """The element offsets of row 1 that a move of `length` positions touches."""
    run = c.run_bytes if length is None or c.position_bytes == 0 else min(length, c.positions) * c.position_bytes
    return sorted(c.row_stride + a * c.outer0_stride + b * c.outer1_stride + i
                  for a in range(c.outer0) for b in range(c.outer1) for i in range(0, run, es))


def _expect(t, dim, length):
    v = t[1] if dim is None or length is None else t[1].narrow(dim - 1, 0, length)
    base, es, out = t.data_ptr(), t.element_size(), []
    off = (v.data_ptr() - base) // es
    idx = torch.cartesian_prod(*(torch.arange(n) for n in v.shape)).reshape(-1, v.dim()) if v.dim() else torch.zeros((1, 0))
    for i in idx.tolist():
        out.append((off + sum(int(a) * s for a, s in zip(i, v.stride()))) * es)
    return sorted(out)


@pytest.mark.parametrize("make,dim", [
    (lambda: torch.zeros((4, 6)), None),
    (lambda: torch.zeros(4, dtype=torch.int64), None),
    (lambda: torch.zeros((4, 6), dtype=torch.uint8), 1),
    (lambda: torch.zeros((4, 2, 5, 3)), 2),
    (lambda: torch.zeros((4, 2, 3, 5)), 3),
    (lambda: torch.zeros((4, 5, 2, 3)), 1),
    (lambda: torch.zeros((4, 3, 8, 6))[:, :, 1:6, 2:5], None),
    (lambda: torch.zeros((5, 4, 3)).transpose(0, 1), None),
    (lambda: torch.zeros((4, 2, 5, 3))[:, 1:], 2),
    (lambda: torch.zeros((4, 2, 5, 3))[:, :, :4], 2),
])
def test_runs_cover_the_state(make, dim):
    t = make()
    c = beam._describe(t, 4, dim)
    assert _elements(c, 4, t.element_size()) == _expect(t, None, None)
    if dim is not None:
        assert c.positions == t.shape[dim]
        for n in (0, 1, t.shape[dim] - 1):
            assert _elements(c, 4, t.element_size(), n) == _expect(t, dim, n)


def test_states_that_are_refused():
    z = torch.zeros
    with pytest.raises(RuntimeError, match="4 rows"):
        beam._describe(z((5, 2)), 4, None)
    with pytest.raises(RuntimeError, match="overlaps itself"):
        beam._describe(z((1, 8)).expand(4, 8), 4, None)
    with pytest.raises(RuntimeError, match="overlaps itself"):
        beam._describe(torch.as_strided(z(64), (4, 8), (4, 1)), 4, None)
    with pytest.raises(RuntimeError, match="more than two strided"):
        beam._describe(z((4, 4, 4, 4, 4))[:, :3, :3, :3, :3], 4, None)
    with pytest.raises(RuntimeError, match="not contiguous"):
        beam._describe(z((4, 5, 8))[:, :, :6], 4, 1)
    with pytest.raises(RuntimeError, match="not contiguous"):
        beam._describe(z((4, 3, 5)).transpose(1, 2), 4, 1)
    with pytest.raises(RuntimeError, match="length dimension"):
        beam._describe(z((4, 5)), 4, 0)
    with pytest.raises(RuntimeError, match="no values"):
        beam._describe(z((4, 0)), 4, None)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        beam.BeamStates([z((4, 2))], 2, 2)
    with pytest.raises(RuntimeError, match="at least one"):
        beam.BeamStates([], 2, 2)
    with pytest.raises(RuntimeError, match="beams"):
        beam.BeamStates([z((66, 2))], 2, 33)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        beam.beam_select(z((1, 2, 8)), z((1, 2)))


def test_bad_arguments_are_errors_before_any_device_call(lib):
    one = 256                                              # an address that is never read
    sel = lib.nsm_beam_select

    def call(logits=one, dt=0, bs=8, ws_=4, scores=one, B=1, W=2, V=8, k=4, pad=0, ws=one):
        return sel(logits, dt, bs, ws_, scores, None, B, W, V, k, pad, one, one, one, ws, 1 << 20, None)

    bad, big = _lib.NSM_ERR_INVALID_ARG, _lib.NSM_ERR_UNSUPPORTED
    assert call(dt=3) == bad and call(logits=None) == bad and call(scores=None) == bad and call(ws=None) == bad
    assert call(B=-1) == bad and call(pad=8) == bad and call(pad=-1) == bad and call(bs=-8) == bad
    assert call(logits=one + 2) == bad
    assert call(W=33) == big and call(k=65) == big and call(V=0) == big and call(k=0) == big
    assert call(B=0) == _lib.NSM_OK
    assert lib.nsm_beam_select_workspace_bytes(1, 33, 8, 4) == 0
    assert lib.nsm_beam_states_bytes(3) == 3 * 72 and lib.nsm_beam_states_bytes(0) == 0
    st = (_lib.BeamStateC * 1)(_lib.BeamStateC(one, 8, 1, 0, 1, 0, 8, 0, 0))
    assert lib.nsm_beam_states_set(st, 1, one, 8, None) == _lib.NSM_ERR_WORKSPACE
    assert lib.nsm_beam_states_set(st, 0, one, 72, None) == bad
    for field, value in (("data", None), ("outer0", 0), ("run_bytes", 0), ("row_stride", -1), ("position_bytes", 3)):
        keep = getattr(st[0], field)
        setattr(st[0], field, value)
        assert lib.nsm_beam_states_set(st, 1, one, 72, None) == bad
        setattr(st[0], field, keep)
    re = lib.nsm_beam_reorder
    assert re(st, one, 1, -1, 2, one, -1, None) == bad
    assert re(st, None, 1, 1, 2, one, -1, None) == bad
    assert re(st, one, 1, 1, 2, None, -1, None) == bad
    assert re(st, one, 1, 1, 33, one, -1, None) == big
    assert re(st, one, 1, 0, 2, one, -1, None) == _lib.NSM_OK


def test_a_state_given_twice_is_refused():
    t = torch.zeros((4, 6))
    beam._check_apart([t, torch.zeros((4, 6)), t[:, 3:]])
    with pytest.raises(RuntimeError, match="must not overlap"):
        beam._check_apart([t, torch.zeros((4, 6)), t])
    with pytest.raises(RuntimeError, match="must not overlap"):
        beam._check_apart([t, t[:, :3]])


def _check(states, rows=4):
    beam._check_disjoint([beam._describe(t, rows, d) for t, d in states], rows)


def test_states_that_share_memory_are_refused():
    z = torch.zeros
    t, kv, cache = z((4, 6)), z((4, 2, 3, 5, 8)), z((4, 3, 2, 5, 8))
    # parts of a buffer side by side, or in between each other, in any order
    _check([(t[:, 3:], None), (z((4, 6)), None), (t[:, :3], 1)])
    _check([(kv[:, 0], 2), (kv[:, 1], 2)])
    _check([(cache[:, :, 1], 2), (cache[:, :, 0], 2)])
    _check([(z((8, 5))[:4], None), (z((8, 5))[4:], None)])
    _check([(t[:, 0], None), (t[:, 2], None), (t[:, 1], None), (t[:, 3:], 1)])
    whole = z(96)
    _check([(whole[:48].view(4, 12)[:, :6], None), (whole[48:].view(4, 12), None)])
    _check([(t[:1, :3], None), (t[:1, 3:], None)], rows=1)
    for states in ([(t, None), (t[:, 3:], None)], [(t[:, 3:], 1), (z((4, 6)), None), (t, 1)],
                   [(t[:, :4], None), (t[:, 3:], None)], [(kv, None), (kv[:, 1], 2)],
                   [(cache[:, :, 1], 2), (cache[:, 1:], None)], [(whole[:48].view(4, 12), None), (whole[44:92].view(4, 12), None)],
                   [(whole[:24].view(4, 6), None), (z((4, 6)), None), (whole.view(torch.uint8)[93:97].view(4, 1), None)]):
        with pytest.raises(RuntimeError, match="share memory"):
            _check(states)
    with pytest.raises(RuntimeError, match="share memory"):
        _check([(t[:1], None), (t[:1, 5:], None)], rows=1)


def test_shared_memory_is_found_run_by_run():
    """Random parts of one buffer: refused where an element belongs to two of them, and only there."""
    gen = torch.Generator().manual_seed(7)
    pick = lambda n: int(torch.randint(0, n, (1,), generator=gen))  # noqa: E731
    seen = [0, 0]
    for _ in range(400):
        shape = [4, 1 + pick(4), 1 + pick(4), 1 + pick(6)]
        order = [0, 1, 2, 3] if pick(3) else [1, 0, 2, 3]
        buf = torch.arange(4 * shape[1] * shape[2] * shape[3]).reshape([shape[i] for i in order]).permute(order)
        states = []
        for _ in range(2 + pick(2)):
            cut = [slice(None)]
            for n in buf.shape[1:]:
                a = pick(n)
                cut.append(slice(a, a + 1 + pick(n - a)))
            states.append(buf[tuple(cut)])
        used = torch.cat([s.reshape(-1) for s in states])
        shared = used.unique().numel() != used.numel()
        seen[shared] += 1
        if shared:
            with pytest.raises(RuntimeError, match="share memory"):
                _check([(s, None) for s in states])
        else:
            _check([(s, None) for s in states])
    assert min(seen) > 40


def test_large_interleaved_states_are_checked_at_once():
    """The keys and values of one buffer, in between each other at every position: not looked through
    one by one (2^26 of them)."""
    data, es, rows, heads, positions, dim = 1 << 40, 2, 256, 64, 4096, 128
    one = [_lib.BeamStateC(data + part * dim * es, heads * positions * 2 * dim * es, 1, 0, heads * positions, 2 * dim * es,
                           dim * es, 0, 0) for part in range(2)]
    beam._check_disjoint(one, rows)
    one[1].data -= 2
    with pytest.raises(RuntimeError, match="share memory"):
        beam._check_disjoint(one, rows)
