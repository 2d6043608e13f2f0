"""The decode-tail example: its operators together, against their definitions
in 64 bits and through a captured graph."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_tail.py")


def _example():
    spec = importlib.util.spec_from_file_location("decode_tail", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _unpack(q, s, z, group):
    codes = torch.stack((q & 15, q >> 4), -1).flatten(-2).double()
    zero = 8.0 if z is None else z.double().repeat_interleave(group, -1)
    return (codes - zero) * s.double().repeat_interleave(group, -1)


def _matrix(w, second):
    d, s, z = (w.w2, w.s2, w.z2) if second else (w.w13, w.s13, w.z13)
    if d.dtype == torch.uint8:
        return _unpack(d, s, z, 64)
    if s is None:
        return d.double()
    return d.double() * s.double().repeat_interleave(128, -2).repeat_interleave(128, -1)[..., :d.shape[-2], :d.shape[-1]]


def _mlp(w, x, e=None):
    w13, w2 = (_matrix(w, b) if e is None else _matrix(w, b)[e] for b in (False, True))
    gate, up = (x @ w13.T).chunk(2, -1)
    return (gate * torch.sigmoid(gate) * up) @ w2.T


def _scores(t):
    """``DecodeTail.scores`` from the definitions, without roundings."""
    rows, vocab = t.logits.shape
    out = torch.empty((rows, vocab), device="cuda", dtype=torch.float64)
    for r in range(rows):
        ids = t.token_ids[r, : t.seq_lens[r]].tolist()
        x = t.embedding[ids[-1]].double()
        p = torch.sigmoid(t.router.double() @ x)
        chosen = torch.topk(p + t.router_bias.double(), t.top_k).indices
        y = _mlp(t.shared, x)
        for e in chosen.tolist():
            y = y + 2.5 * p[e] / p[chosen].sum() * _mlp(t.experts, x, e)
        x = _unpack(t.vocab_q, t.vocab_s, None, 128) @ (x + y)
        x[7] += 0.5
        for v in set(ids):
            x[v] = x[v] / t.repetition[r].double() if x[v] > 0 else x[v] * t.repetition[r].double()
            n = ids[int(t.prompt_lens[r]):].count(v)
            if n:
                x[v] -= t.frequency[r].double() * n + t.presence[r].double()
        bits = t.allowed[r].cpu().unsqueeze(1) >> torch.arange(32, dtype=torch.int32) & 1
        x[bits.flatten()[:vocab].cuda() == 0] = -torch.inf
        out[r] = x
    return out


@pytest.mark.parametrize("weights", ["bf16", "fp8", "w4"])
def test_scores_are_the_definitions(weights):
    t = _example().DecodeTail(requests=3, hidden=256, experts=12, top_k=3, inner=128, shared=256, vocab=1003, max_len=20,
                              weights=weights)
    t.forbid(1, [5, 31, 32, 1002])
    for _ in range(4):
        t.step()
    got, ref = t.scores().double(), _scores(t)
    assert torch.equal(torch.isinf(got), torch.isinf(ref)) and (ref[1, [5, 31, 32, 1002]] == -torch.inf).all()
    ok = torch.isfinite(ref)
    # a logit's own bf16 rounding before its penalties and after, and those of
    # x and the layer: 2^-8 each of values of size |x| ~ 4 through unit rows
    assert ((got - ref).abs() <= 2 * 2.0 ** -8 * ref.abs() + 6 * 2.0 ** -8 * 4)[ok].all()


def test_graph_steps_are_eager_steps_and_masks_hold():
    module = _example()
    make = dict(requests=5, hidden=512, experts=16, top_k=2, inner=256, shared=256, vocab=4000, max_len=40)
    a, b = module.DecodeTail(**make), module.DecodeTail(**make)
    for t in (a, b):
        t.presence.fill_(100.0)  # no token a second time
        t.forbid(2, range(0, 4000, 2))
    graph = b.capture()
    for _ in range(30):
        a.step()
        graph.replay()
    assert torch.equal(a.token_ids, b.token_ids) and torch.equal(a.seq_lens, b.seq_lens)
    for row in a.token_ids[:, 1:31].tolist():
        assert len(set(row)) == 30 and min(row) >= 0
    assert (a.token_ids[2, 1:31] % 2 == 1).all()


def test_main_runs(capsys):
    answers = _example().main(["--requests", "2", "--steps", "6", "--vocab", "2048"])
    assert [len(a) for a in answers] == [6, 6]
    assert "us a step" in capsys.readouterr().out


@pytest.mark.parametrize("captured", [False, True])
def test_steps_past_a_full_history_stay_inside_it(captured):
    t = _example().DecodeTail(requests=3, hidden=256, experts=8, top_k=2, inner=128, shared=128, vocab=600, max_len=4)
    step = t.capture().replay if captured else t.step
    for _ in range(3):
        step()
    assert t.seq_lens.tolist() == [4] * 3
    full = t.token_ids.clone()
    for _ in range(5):
        step()
    assert t.seq_lens.tolist() == [4] * 3 and torch.equal(t.token_ids[:, :3], full[:, :3])
    assert ((t.token_ids >= 0) & (t.token_ids < 600)).all()


def test_main_without_steps():
    assert _example().main(["--requests", "2", "--steps", "0", "--vocab", "2048"]) == [[], []]
