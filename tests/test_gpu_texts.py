"""Stages that follow different texts on the GPU: the text cross-attention of
kernels.cross_attention against the masked torch path, through forward_stages
and through the wavefront engine."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(texts, lens, seed=0):
    from waveforcing_b200.wavefront.dit import DiTConfig, WanDiT

    dev = torch.device("cuda", 0)
    cfg = DiTConfig(dim=256, heads=2, layers=2, ffn=512, text_len=16, text_dim=64, lat_h=16, lat_w=24)
    model = WanDiT.random(cfg, dev, seed=seed)
    g = torch.Generator().manual_seed(1)
    text = torch.randn((3, cfg.text_len, cfg.text_dim), generator=g).to(dev)
    model.set_text(text if texts else text[0], lens)
    return model, dev


def _cos(a, b):
    return torch.nn.functional.cosine_similarity(a.flatten().double(), b.flatten().double(), dim=0).item()


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("lens", [None, [16, 5, 0]])
def test_forward_matches_the_torch_path(fused, lens):
    from waveforcing_b200.runtime import backend
    from waveforcing_b200.wavefront.dit import StageTask

    model, dev = _model(True, lens)
    g = torch.Generator().manual_seed(2)
    x = torch.randn((3, model.cfg.in_ch, model.cfg.frames_per_block, 16, 24), generator=g).to(dev)
    tasks = [StageTask(x[i], 600.0, 3 * i, 2 - i, text=n, kv_only=i == 0) for i, n in enumerate([1, 2, 1])]
    out = {}
    for name in ("wf_b200", "torch_sdpa"):
        backend.select_backend(name)
        out[name] = model.forward_stages(tasks, fused=fused)
    assert out["wf_b200"][0] is None
    for a, b in zip(out["wf_b200"][1:], out["torch_sdpa"][1:]):
        assert torch.isfinite(a).all() and _cos(a, b) >= 0.999


def _run(name, several, texts=(), num_frames=18):
    from waveforcing_b200.runtime import backend
    from waveforcing_b200.wavefront.engine import EngineConfig, WavefrontEngine

    backend.select_backend(name)
    model, dev = _model(several, [16, 9, 4] if several else None)
    eng = WavefrontEngine(model, EngineConfig(num_frames=num_frames, texts=texts), device=dev)
    for t in range(eng.num_ticks):
        eng.tick(t)
    torch.cuda.synchronize()
    out = torch.cat([eng.final[c].float() for c in sorted(eng.final)], dim=1)
    eng.close()
    return out


def test_engine_changes_texts_along_the_chunks():
    texts = (0, 0, 1, 2)
    a, b = _run("wf_b200", True, texts), _run("torch_sdpa", True, texts)
    assert torch.isfinite(a).all() and _cos(a, b) >= 0.999
    # one text of several is that text alone
    assert _cos(_run("wf_b200", True, (0,)), _run("wf_b200", False)) >= 0.999


def test_a_new_list_of_texts_does_not_wait_for_the_device():
    from waveforcing_b200.wavefront.dit import StageTask

    model, dev = _model(True, [16, 5, 0])
    tasks = [[StageTask(None, 600.0, 0, 0, text=n) for n in texts] for texts in ([0, 1], [2, 2, 1], [1])]
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = [model._text_index(t) for t in tasks]
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert [g.tolist() for g in got] == [[0, 1], [2, 2, 1], [1]] and all(g.dtype == torch.int32 for g in got)
