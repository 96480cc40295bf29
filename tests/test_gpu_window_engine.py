"""The engine with an attention window (sinks + sliding window in every layer, prompt chunks and decode steps in their CUDA
graphs) against a plain FP32 forward of the same model with that mask, and its cache held to the window's pages."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from redline_llm_b200.engine import Engine, ModelConfig, ModelWeights  # noqa: E402

CFG = ModelConfig(layers=2, hidden=256, inter=512, q_heads=6, kv_heads=2, head_dim=128, vocab=1000, rope_theta=1e4,
                  eos_token_id=999)


@pytest.fixture(scope="module")
def weights():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return ModelWeights(CFG, torch.device("cuda", 0), seed=21, std=0.08)


def forward(w, ids, window, sinks):
    c = CFG
    x = w.embed.float()[torch.tensor(ids, device="cuda")]
    t = len(ids)
    pos = torch.arange(t, device="cuda")
    inv = 1.0 / (c.rope_theta ** (torch.arange(0, c.head_dim, 2, device="cuda", dtype=torch.float64) / c.head_dim))
    ang = pos.double()[:, None] * inv[None]
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

    def norm(v, wt):
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + c.eps) * wt.float()

    def rope(v):
        a, b = v[..., :c.head_dim // 2], v[..., c.head_dim // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    k_pos, q_pos = pos[None, :], pos[:, None]
    seen = (k_pos <= q_pos) & ((k_pos < sinks) | (k_pos > q_pos - window))
    for L in w.layers:
        qkv = norm(x, L["in_norm"]) @ L["qkv"].float().t() + L["qkv_bias"].float()
        q = rope(qkv[:, :c.q_width].view(t, c.q_heads, c.head_dim))
        k = rope(qkv[:, c.q_width:c.q_width + c.kv_width].view(t, c.kv_heads, c.head_dim))
        v = qkv[:, c.q_width + c.kv_width:].view(t, c.kv_heads, c.head_dim)
        g = c.q_heads // c.kv_heads
        s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(g, 1)) / c.head_dim ** 0.5
        p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
        x = x + torch.einsum("hqk,khd->qhd", p, v.repeat_interleave(g, 1)).reshape(t, -1) @ L["o"].float().t()
        gu = norm(x, L["post_norm"]) @ L["gate_up"].float().t()
        x = x + (torch.nn.functional.silu(gu[:, :c.inter]) * gu[:, c.inter:]) @ L["down"].float().t()
    return norm(x, w.final_norm) @ w.lm_head.float().t()


@pytest.mark.parametrize("graphs,window,sinks", [(True, 48, 4), (False, 33, 0), (True, 200, 20)])
def test_logits_of_every_decode_step(weights, graphs, window, sinks):
    """Teacher-forced, two requests of different lengths, the prompt in chunks: each decode step's logits against the FP32
    forward with the same mask. The model rounds to FP16 between its stages, so the bound is a fraction of the logits'
    range, as for the engine without a window; a mask off by one page moves them by several times as much."""
    rng = np.random.default_rng(window)
    prompts = [rng.integers(0, 998, n).tolist() for n in (150, 61)]
    forced = [rng.integers(0, 998, 40).tolist() for _ in prompts]
    e = Engine(kv_pool_gb=0.02, max_batch=2, max_seq_len=512, prefill_chunk=32, config=CFG, weights=weights,
               enable_cuda_graphs=graphs, attention_window=window, attention_sinks=sinks, device_feedback=False)
    ids = [e.add_request(p, len(f), ignore_eos=True, forced_tokens=f) for p, f in zip(prompts, forced)]
    want = [forward(weights, p + f, window, sinks) for p, f in zip(prompts, forced)]
    full = forward(weights, prompts[0] + forced[0], 10**6, 0)
    scale = float(want[0].abs().max())
    worst = 0.0
    while e.stats()["running"] or e.stats()["waiting"]:
        before = [(r.req_id, r.cached) for r in e.scheduler.running]
        if len(before) < 2 or any(r.prefilled < len(r.prompt) for r in e.scheduler.running):
            e.step()
            continue
        e.step()
        for i, (rid, cached) in enumerate(before):
            got = e.exec.logits[i].float()
            worst = max(worst, float((got - want[ids.index(rid)][cached]).abs().max()))
    assert worst < 0.03 * scale, worst / scale
    n = len(prompts[0])
    assert float((full[n:n + 39] - want[0][n:n + 39]).abs().max()) > 0.03 * scale or window >= 200, "the window does not matter here"
    assert e.exec.K.window_attention_health(e.exec.window_ws) == 0 and e.exec.K.prefill_attention_health() == 0
    assert e.allocator.free_blocks == e.allocator.total - 1 and e.allocator.reserved == 0


def test_a_request_longer_than_the_pool_runs_in_its_window(weights):
    """A pool of about thirty pages serves a request of 700 tokens whose window and sinks fit it; pipelined steps."""
    block = CFG.block_bytes()
    e = Engine(kv_pool_gb=30 * block / (1 << 30) + 1e-9, max_batch=1, max_seq_len=1024, prefill_chunk=64, config=CFG, weights=weights,
               attention_window=128, attention_sinks=4)
    assert e.allocator.total <= 31
    prompt = np.random.default_rng(1).integers(0, 998, 600).tolist()
    e.add_request(prompt, 100, ignore_eos=True)
    got, most = [], 0
    for _ in range(400):
        got += e.step_pipelined()
        most = max(most, e.allocator.total - 1 - e.allocator.free_blocks)
        if not e.scheduler.running and not e.scheduler.waiting and not e.in_flight:
            break
    got += e.drain()
    assert len(got) == 100 and got[-1][2] and e.scheduler.aborts == 0
    assert most <= e.scheduler.held_blocks() < 40
    e2 = Engine(kv_pool_gb=0.02, max_batch=1, max_seq_len=1024, prefill_chunk=64, config=CFG, weights=weights,
                attention_window=128, attention_sinks=4)
    e2.add_request(prompt, 100, ignore_eos=True)
    want = []
    while e2.scheduler.running or e2.scheduler.waiting:
        want += e2.step()
    assert [t[1] for t in got] == [t[1] for t in want], "pages given back were still in use"


def test_arguments_are_checked():
    for kw in (dict(attention_window=-1), dict(attention_sinks=-1), dict(attention_sinks=4),
               dict(attention_window=64, prefill_attention="composite")):
        with pytest.raises(ValueError):
            Engine(kv_pool_gb=0.01, config=CFG, **kw)
