"""Stages that follow different texts: WanDiT.set_text with several texts, a task's
``text``, the engine's ``texts``, and the masked fallback of the text
cross-attention (CPU).  The kernel's side of it is in test_gpu_texts.py."""
import pytest
import torch

from waveforcing_b200 import kernels
from waveforcing_b200.runtime import backend
from waveforcing_b200.wavefront import dit as D
from waveforcing_b200.wavefront.engine import EngineConfig

CFG = dict(dim=256, heads=2, layers=2, ffn=512, text_len=16, text_dim=64, lat_h=4, lat_w=4)


def _rope(x, cos, sin, out=None):
    re, im = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.stack([re * c - im * s, re * s + im * c], -1).flatten(-2).to(x.dtype)


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(kernels, "rope_apply", _rope)
    monkeypatch.setitem(backend._WAVE_STATE, "attn", "torch_sdpa")
    m = D.WanDiT.random(D.DiTConfig(**CFG), torch.device("cpu"), dtype=torch.float32, seed=0)
    g = torch.Generator().manual_seed(1)
    m._test_texts = torch.randn((3, 16, 64), generator=g)
    m._test_latents = torch.randn((4, m.cfg.in_ch, m.cfg.frames_per_block, 4, 4), generator=g)
    return m


def _tasks(m, texts, kv_only=()):
    return [D.StageTask(m._test_latents[i], 600.0, 3 * i, 3 - i, kv_only=i in kv_only, text=n)
            for i, n in enumerate(texts)]


def test_tasks_follow_their_own_texts(model):
    lens, texts = [16, 5, 1], [2, 0, 1, 1]
    model.set_text(model._test_texts, lens)
    got = model.forward_stages(_tasks(model, texts), fused=False)
    for i, n in enumerate(texts):
        model.set_text(model._test_texts[n, :lens[n]])
        task = _tasks(model, [0] * 4)[i]
        want = model.forward_stages([task], fused=False)[0]
        # f32 throughout: sums of at most 512 terms in another order
        assert torch.allclose(got[i], want, rtol=0, atol=512 * 2.0 ** -24 * 8 * want.abs().max().item())


def test_kv_only_tasks_leave_the_others_their_texts(model):
    model.set_text(model._test_texts, [16, 5, 1])
    every = model.forward_stages(_tasks(model, [1, 2, 0]), fused=False)
    some = model.forward_stages(_tasks(model, [1, 2, 0], kv_only=(1,)), fused=False)
    assert some[1] is None
    for i in (0, 2):
        assert torch.allclose(some[i], every[i], rtol=0, atol=512 * 2.0 ** -24 * 8 * every[i].abs().max().item())


def test_an_empty_text_adds_nothing(model):
    q, kv = torch.randn(2, 3, 2, 128), torch.randn(2, 4, 2, 128)
    index = torch.tensor([1, 0], dtype=torch.int32)
    o = backend.cross_attention(q, kv, kv, index, torch.tensor([4, 0], dtype=torch.int32))
    assert (o[0] == 0).all() and torch.isfinite(o[1]).all() and (o[1] != 0).any()


@pytest.mark.parametrize("text, lens", [((16, 64), [16]), ((3, 16, 64), [16, 5]), ((3, 16, 64), [16, 17, 1]),
                                        ((3, 16, 64), [16, -1, 1]), ((64,), None)])
def test_set_text_refuses(model, text, lens):
    with pytest.raises(ValueError, match="set_text"):
        model.set_text(torch.zeros(text), lens)


@pytest.mark.parametrize("several, text", [(False, 1), (True, 3), (True, -1)])
def test_tasks_of_texts_that_were_not_given_are_refused(model, several, text):
    model.set_text(model._test_texts if several else model._test_texts[0])
    with pytest.raises(ValueError, match="texts"):
        model.forward_stages(_tasks(model, [text]), fused=False)


def test_engine_chunks_follow_the_last_text_from_then_on():
    cfg = EngineConfig(texts=(0, 0, 2, 1))
    assert [cfg.text_of(c) for c in range(6)] == [0, 0, 2, 1, 1, 1]
    assert EngineConfig().text_of(5) == 0


def test_lists_of_texts_leave_nothing_behind(model):
    """A text per chunk gives a new list every tick."""
    model.set_text(model._test_texts)
    kept = lambda: {k: len(v) for k, v in vars(model).items() if hasattr(v, "__len__")}  # noqa: E731
    model.forward_stages(_tasks(model, [0, 0, 0]), fused=False)
    before = kept()
    for n in range(27):
        model.forward_stages(_tasks(model, [n // 9, n // 3 % 3, n % 3]), fused=False)
    assert kept() == before
