"""Beam search around the decode path: the best continuations of several beams
(``beam_select``), their states put in order (``BeamStates``), and a step that
joins them with a head (``BeamSearch``).

The reference decodes one sequence; a batch of beams goes through this build's
multi-row entries (``route_sparse_mlp``, ``union_decode``: beams of one prompt
share most of their blocks), a head (``Nf4LmHead``, ``Linear4bit``) and these.
"""
from __future__ import annotations

import torch

from . import _lib
from ._torch import dtype_code, require_cuda, stream_handle

MAX_BEAMS, MAX_CANDIDATES = 32, 64


def beam_select(logits: torch.Tensor, scores: torch.Tensor, *, num_candidates: int | None = None,
                finished: torch.Tensor | None = None, pad_token: int = 0):
    """``(scores fp32, tokens int64, parents int64)``, each ``[batch,
    num_candidates]``: for each batch item the best (beam, token) by ``scores +
    log_softmax(logits)``, best first, equal ones in the order of beam, then token.

    ``logits [batch, beams, vocab]`` or ``[batch * beams, vocab]`` (fp32 / fp16 /
    bf16; a view into a wider buffer is read in place), ``scores [batch,
    beams]`` fp32 (-infinity: the beam is out).  ``num_candidates``: default twice
    the beams.  ``finished [batch, beams]`` (bool): such a beam is one candidate,
    ``pad_token`` at its own score.  A logit of -infinity or NaN is no
    candidate; where too few exist: score -infinity, token -1, parent 0.
    Scores are formed and compared in 64 bits, with log-sum-exps of fp32 sums.  (In a
    row of nothing but the type's lowest value 64 bits lose the logarithm of the sum: its words
    have the beam's own score.  Mask with -infinity what may not come.)"""
    require_cuda(logits, "logits")
    dev = logits.device
    if scores.dim() != 2 or scores.dtype != torch.float32 or scores.device != dev:
        raise RuntimeError(f"scores must be fp32 [batch, beams] on {dev}, got {tuple(scores.shape)} {scores.dtype} "
                           f"on {scores.device}")
    B, W = scores.shape
    if logits.dim() == 2 and logits.shape[0] == B * W:
        logits = logits.unflatten(0, (B, W)) if B * W else logits.reshape(B, W, logits.shape[1])
    if logits.dim() != 3 or logits.shape[0] != B or logits.shape[1] != W:
        raise RuntimeError(f"logits has shape {tuple(logits.shape)} for scores of {tuple(scores.shape)}")
    V = logits.shape[2]
    k = 2 * W if num_candidates is None else int(num_candidates)
    if not 1 <= W <= MAX_BEAMS or not 1 <= k <= MAX_CANDIDATES or V < 1:
        raise RuntimeError(f"beam_select takes 1 to {MAX_BEAMS} beams, 1 to {MAX_CANDIDATES} candidates and a "
                           f"vocabulary, got {W} beams, {k} candidates and {V} tokens")
    if not 0 <= pad_token < V:
        raise RuntimeError(f"pad_token ({pad_token}) is outside the vocabulary of {V}")
    code = dtype_code(logits.dtype)
    fin = None
    if finished is not None:
        if finished.shape != scores.shape or finished.dtype not in (torch.bool, torch.uint8) or finished.device != dev:
            raise RuntimeError(f"finished must be bool {tuple(scores.shape)} on {dev}")
        finished = finished.contiguous()
        fin = finished.data_ptr()
    if logits.stride(2) != 1 and V > 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _select(logits, code, scores, fin, B, W, V, k, pad_token, dev)
    return _select(logits, code, scores, fin, B, W, V, k, pad_token, dev)


_WS_BYTES: dict[tuple[int, int, int, int, int], int] = {}  # by device and sizes
_LIB = None


def _select(logits, code, scores, fin, B, W, V, k, pad_token, dev):
    global _LIB
    lib = _LIB
    if lib is None:
        lib = _LIB = _lib.load()
    out_s = torch.empty(B, k, dtype=torch.float32, device=dev)
    out_t = torch.empty(B, k, dtype=torch.int64, device=dev)
    out_p = torch.empty_like(out_t)
    if B:
        key = (dev.index, B, W, V, k)
        need = _WS_BYTES.get(key)
        if need is None:
            if len(_WS_BYTES) > 4096:
                _WS_BYTES.clear()
            need = _WS_BYTES[key] = int(lib.nsm_beam_select_workspace_bytes(B, W, V, k))
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else out_s  # (a pointer that is not used)
        stride = logits.stride()
        status = lib.nsm_beam_select(logits.data_ptr(), code, stride[0], stride[1], scores.data_ptr(), fin, B, W, V, k,
                                     pad_token, out_s.data_ptr(), out_t.data_ptr(), out_p.data_ptr(), ws.data_ptr(),
                                     need, stream_handle(dev))
        if status:
            _lib.check(status, "nsm_beam_select")
    return out_s, out_t, out_p


def _describe(t: torch.Tensor, rows: int, length_dim: int | None) -> _lib.BeamStateC:
    """The runs of one state ``[rows, ...]``: trailing contiguous dimensions are a
    run (from the positions on, when there are), the others in between at most two
    strided ones."""
    es = t.element_size()
    if t.dim() < 1 or t.shape[0] != rows:
        raise RuntimeError(f"a state has shape {tuple(t.shape)} but there are {rows} rows (batch * beams)")
    if length_dim is not None:
        length_dim = length_dim + t.dim() if length_dim < 0 else length_dim
        if not 1 <= length_dim < t.dim():
            raise RuntimeError(f"length dimension {length_dim} of a state of shape {tuple(t.shape)}")
    if t.numel() == 0:
        raise RuntimeError(f"a state of shape {tuple(t.shape)} has no values")
    # no two elements may share memory
    span = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda e: e[1]):
        if s < span:
            raise RuntimeError(f"a state of shape {tuple(t.shape)} and strides {t.stride()} overlaps itself")
        span = (n - 1) * s + span
    dims = [(n, s) for n, s in zip(t.shape[1:], t.stride()[1:])]
    tail = len(dims) if length_dim is None else length_dim  # dims[tail:] lie inside a position
    inner = 1
    if length_dim is not None:
        for n, s in reversed(dims[tail:]):
            if n > 1 and s != inner:
                raise RuntimeError(f"positions of a state of strides {t.stride()} are not contiguous")
            inner *= n
        count, step = dims[tail - 1]
        if count > 1 and step != inner:
            raise RuntimeError(f"positions of a state of strides {t.stride()} are not contiguous")
        run, rest = inner * count, dims[:tail - 1]
    else:
        run, rest = 1, list(dims)
        while rest and (rest[-1][0] == 1 or rest[-1][1] == run):
            run *= rest.pop()[0]
        count = 0
    outer: list[tuple[int, int]] = []
    for n, s in rest:
        if n == 1:
            continue
        if outer and outer[-1][1] == n * s:
            outer[-1] = (outer[-1][0] * n, s)
        else:
            outer.append((n, s))
    if len(outer) > 2:
        raise RuntimeError(f"a state of shape {tuple(t.shape)} and strides {t.stride()} has more than two strided "
                           "dimensions")
    (o0, s0), (o1, s1) = ([(1, 0)] * 2 + outer)[-2:]
    return _lib.BeamStateC(t.data_ptr(), t.stride(0) * es if rows > 1 else 0, o0, s0 * es, o1, s1 * es, run * es,
                           inner * es if length_dim is not None else 0, count)


def _check_apart(states) -> None:
    """No state is given twice: it would be put in order twice, at the same time."""
    first = [t.data_ptr() for t in states]
    if len(set(first)) != len(first):
        raise RuntimeError("two states begin at the same address: states must not overlap")


def _check_disjoint(described, rows: int) -> None:
    """No byte belongs to two states: different states move at the same time.  States whose
    extents meet are compared run by run, so that parts of one buffer may lie in between
    each other."""
    # where a state begins, its run, and the (count, stride) of its rows and outer dimensions
    sets = [(c.data, c.run_bytes, [(n, s) for n, s in ((rows, c.row_stride), (c.outer0, c.outer0_stride),
                                                       (c.outer1, c.outer1_stride)) if n > 1]) for c in described]

    def end(e):
        return e[0] + e[1] + sum((n - 1) * s for n, s in e[2])

    meeting: list[list] = []
    reach = 0
    for e in sorted(sets, key=lambda e: e[0]):
        if e[0] >= reach:
            meeting.append([])
        meeting[-1].append(e)
        reach = max(reach, end(e))
    for group in meeting:
        if len(group) < 2:
            continue
        # A stride that all have, and that all of them fit into without it: what lies at different
        # multiples of it is apart, and one multiple is as the others.
        again = True
        while again:
            again = False
            for step in {s for _, s in group[0][2]}:
                if all(any(s == step for _, s in e[2]) for e in group):
                    rest = [(at, run, [d for d in dims if d[1] != step]) for at, run, dims in group]
                    if max(end(e) for e in rest) - min(e[0] for e in rest) <= step:
                        group, again = rest, True
                        break
        starts, ends = [], []
        for at, run, dims in group:
            first = torch.tensor([at], dtype=torch.int64)
            for n, s in dims:
                first = (first[:, None] + torch.arange(n, dtype=torch.int64) * s).reshape(-1)
            starts.append(first)
            ends.append(first + run)
        first, order = torch.cat(starts).sort()
        if bool((first[1:] < torch.cat(ends)[order][:-1]).any()):
            raise RuntimeError("two states share memory: states must not overlap")


class BeamStates:
    """The per-beam states of a decode (caches, histories, residuals), reordered in
    place and in one launch after each selection.

    ``states``: CUDA tensors ``[batch * beams, ...]`` of any type, row ``b *
    beams + w`` beam ``w`` of item ``b``; they are kept, must keep their memory
    and must not overlap (states that share a byte are refused).  ``length_dims``: for each
    state the dimension that holds positions, or ``None``; :meth:`reorder_` can then move the first ``length`` positions only."""

    def __init__(self, states, batch: int, beams: int, length_dims=None):
        self.states = list(states)
        self.batch, self.beams = int(batch), int(beams)
        if self.batch < 1 or not 1 <= self.beams <= MAX_BEAMS:
            raise RuntimeError(f"BeamStates takes 1 to {MAX_BEAMS} beams, got batch {batch} and {beams} beams")
        if not self.states:
            raise RuntimeError("BeamStates needs at least one state")
        dims = [None] * len(self.states) if length_dims is None else list(length_dims)
        if len(dims) != len(self.states):
            raise RuntimeError(f"{len(dims)} length dimensions for {len(self.states)} states")
        for t in self.states:
            require_cuda(t, "a state")
            if t.device != self.states[0].device:
                raise RuntimeError(f"states are on {self.states[0].device} and {t.device}")
        _check_apart(self.states)
        self.device = self.states[0].device
        n = len(self.states)
        described = [_describe(t, self.batch * self.beams, d) for t, d in zip(self.states, dims)]
        _check_disjoint(described, self.batch * self.beams)
        self._c = (_lib.BeamStateC * n)(*described)
        self.max_length = min((c.positions for c in self._c if c.position_bytes), default=None)
        self._lib = lib = _lib.load()
        with torch.cuda.device(self.device):
            self._table = torch.empty(int(lib.nsm_beam_states_bytes(n)), dtype=torch.uint8, device=self.device)
            _lib.check(lib.nsm_beam_states_set(self._c, n, self._table.data_ptr(), self._table.numel(),
                                               stream_handle(self.device)), "nsm_beam_states_set")

    def reorder_(self, parents: torch.Tensor, length: int | None = None) -> None:
        """``state[b, w] = state[b, parents[b, w]]`` for every state (``parents``
        int64 ``[batch, beams]``; a value outside ``0 .. beams - 1`` leaves its
        row as it is)."""
        if parents.dtype != torch.int64 or parents.numel() != self.batch * self.beams or parents.device != self.device:
            raise RuntimeError(f"parents must be int64 [{self.batch}, {self.beams}] on {self.device}, got "
                               f"{tuple(parents.shape)} {parents.dtype} on {parents.device}")
        if length is not None and (length < 0 or self.max_length is None or length > self.max_length):
            raise RuntimeError(f"length {length} is outside the states' {self.max_length} positions")
        parents = parents.contiguous()
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                self._run(parents, length)
        else:
            self._run(parents, length)

    def _run(self, parents: torch.Tensor, length: int | None) -> None:
        _lib.check(self._lib.nsm_beam_reorder(self._c, self._table.data_ptr(), len(self.states), self.batch, self.beams,
                                              parents.data_ptr(), -1 if length is None else length,
                                              stream_handle(self.device)), "nsm_beam_reorder")


class BeamSearch:
    """Beam search over a head: each :meth:`step` takes the beams' hidden states,
    keeps the ``beams`` best continuations of each prompt and puts every state in
    their order.  Finished beams (``eos_token`` chosen) stay at their score.

    ``head``: ``head(hidden, out_dtype)`` -> logits (``Nf4LmHead``, ``Linear4bit``).
    ``states`` / ``length_dims``: the caller's own states, as in ``BeamStates``."""

    def __init__(self, head, batch: int, beams: int, *, max_tokens: int, eos_token: int | None = None,
                 pad_token: int = 0, states=(), length_dims=None, logits_dtype: torch.dtype = torch.float32):
        self.head, self.batch, self.beams = head, int(batch), int(beams)
        self.eos_token, self.pad_token, self.logits_dtype = eos_token, int(pad_token), logits_dtype
        dev, rows = head.device, self.batch * self.beams
        if max_tokens < 1:
            raise RuntimeError(f"max_tokens must be positive, got {max_tokens}")
        self.history = torch.full((rows, int(max_tokens)), self.pad_token, dtype=torch.int64, device=dev)
        self._own = BeamStates([self.history], self.batch, self.beams, [1])
        self._states = BeamStates(states, self.batch, self.beams, length_dims) if len(states) else None
        self.scores = torch.empty((self.batch, self.beams), dtype=torch.float32, device=dev)
        self.finished = torch.empty((self.batch, self.beams), dtype=torch.bool, device=dev)
        self.reset()

    def reset(self) -> None:
        """Back to the prompts: only beam 0 of each is alive (its row holds the state
        that all continuations start from)."""
        self.scores.fill_(float("-inf"))
        self.scores[:, 0] = 0.0
        self.finished.zero_()
        self.history.fill_(self.pad_token)
        self.length = 0

    def step(self, hidden: torch.Tensor, length: int | None = None) -> torch.Tensor:
        """``hidden [batch * beams, H]`` (or ``[batch, beams, H]``) -> the next token
        of each beam ``[batch, beams]`` int64; ``length``: positions that the
        caller's states hold so far."""
        if self.length >= self.history.shape[1]:
            raise RuntimeError(f"the history holds {self.history.shape[1]} tokens")
        rows = self.batch * self.beams
        logits = self.head(hidden.reshape(rows, hidden.shape[-1]), self.logits_dtype)
        scores, tokens, parents = beam_select(logits, self.scores, num_candidates=self.beams, finished=self.finished,
                                              pad_token=self.pad_token)
        tokens.masked_fill_(tokens < 0, self.pad_token)  # beams that are out
        if self._states is not None:
            self._states.reorder_(parents, length)
        if self.length:
            self._own.reorder_(parents, self.length)
        self.history[:, self.length] = tokens.reshape(-1)
        finished = torch.gather(self.finished, 1, parents)
        self.finished = finished if self.eos_token is None else finished | (tokens == self.eos_token)
        self.scores = scores
        self.length += 1
        return tokens

    def error(self) -> int:
        """The head's error word, read and cleared (``Linear4bit.error``; 0 for a head that
        has none).  Not 0: logits were NaN, which no candidate comes from, so the tokens since
        the last check are not the best ones.  Synchronises; once after a decode is enough."""
        read = getattr(self.head, "error", None)
        return int(read()) if read is not None else 0

    def sequences(self) -> torch.Tensor:
        """The tokens so far, ``[batch, beams, length]``, best beam first."""
        return self.history.view(self.batch, self.beams, -1)[:, :, :self.length]
