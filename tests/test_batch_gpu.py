"""The operators over key ranges together, as they are used: `LlamaBatch` packs
prompts into one pass, stores each into its slot and steps all sequences at
once. Logits against the CPU restatement of the plain stack and against a dense
64-bit stack with capped, biased and windowed scores and scaled rotary
positions, by the rule of test_stack_gpu.py (the prompts' queries and weights and
the caches are f16: 5e-3 of the logits' scale)."""
from dataclasses import dataclass

import numpy as np
import pytest
import torch

import ranges_ref as ref
from oracle.stack import CpuStack, StackConfig, random_weights
from tests.configs import SEED

pytestmark = pytest.mark.gpu


@dataclass(frozen=True)
class Config(StackConfig):
    rope_dim: int = 0
    rope_interleaved: bool = False
    rope_scaling: tuple | None = None
    softcap: float = 0.0
    window: int = 0
    shared: int = 0
    slopes: tuple | None = None


def near(got, want, what):
    want, got = np.asarray(want, np.float64), np.asarray(got, np.float64)
    scale = np.abs(want).max()
    assert np.abs(want - got).max() < 5e-3 * scale, (what, float(np.abs(want - got).max() / scale))


def prompts_of(cfg, lens, seed=SEED):
    rng = np.random.default_rng(seed)
    return [[int(t) for t in rng.integers(0, cfg.vocab, n)] for n in lens]


def test_packed_prompts_and_steps_decode_like_the_cpu(gpu):
    """Three prompts in one pass, then tokens of all of them and of some, against one CPU stack each."""
    from ttsxabe_amd.stack import LlamaBatch
    cfg = StackConfig()
    w = random_weights(cfg, SEED)
    dev = LlamaBatch(gpu, cfg, w, slots=4, cap=300)
    cpus = [CpuStack(cfg, w) for _ in range(3)]
    prompts, slots = prompts_of(cfg, [70, 1, 255]), [2, 0, 3]
    want = [c.forward(p) for c, p in zip(cpus, prompts)]
    got = dev.prefill(prompts, slots).cpu().numpy()
    for turn in range(8):
        for g, x in zip(got, want):
            near(g, x, turn)
            assert int(g.argmax()) == int(x.argmax())
        live = [0, 1, 2] if turn % 3 else [2, 0]
        ids = [int(want[i].argmax()) for i in live]
        want = [cpus[i].forward([t]) for i, t in zip(live, ids)]
        got = dev.step(ids, [slots[i] for i in live]).cpu().numpy()
        full = [cpus[i].past for i in range(3)]
        assert [dev.length[s] for s in slots] == full
        if len(live) < 3:  # the third sequence catches up
            t = int(np.argmax(np.random.default_rng(turn).random(cfg.vocab)))
            a, b = cpus[1].forward([t]), dev.step([t], [slots[1]]).cpu().numpy()[0]
            near(b, a, turn)
            want, got = [want[1], a, want[0]], np.stack([got[1], b, got[0]])


def test_a_gguf_rotates_as_it_is_stored(gpu, tmp_path):
    """The interleaved rotation of a GGUF's rows is the halves rotation of the unpermuted ones."""
    from ttsxabe_amd.llama_gguf import load_llama_gguf
    from ttsxabe_amd.stack import LlamaBatch, LlamaStack
    from tests.test_gguf import llama_gguf
    cfg = StackConfig()
    llama_gguf(tmp_path / "m.gguf", cfg, random_weights(cfg, SEED + 7),
               rope_freqs=np.linspace(1.0, 8.0, cfg.head_dim // 2, dtype=np.float32))
    plain, wp = load_llama_gguf(tmp_path / "m.gguf")
    inter, wi = load_llama_gguf(tmp_path / "m.gguf", interleaved=True)
    assert inter.rope_interleaved and not plain.rope_interleaved
    assert not np.array_equal(wp["0.wq"], wi["0.wq"])
    with pytest.raises(ValueError):
        LlamaStack(gpu, inter, wi)
    one, two = LlamaBatch(gpu, plain, wp, 2, 128), LlamaBatch(gpu, inter, wi, 2, 128)
    prompts = prompts_of(cfg, [40, 9])
    a, b = one.prefill(prompts, [1, 0]), two.prefill(prompts, [1, 0])
    near(b.cpu(), a.cpu(), "prompt")
    for t in range(3):
        ids = a.argmax(1).tolist()
        a, b = one.step(ids, [1, 0]), two.step(ids, [1, 0])
        near(b.cpu(), a.cpu(), t)


def dense(cfg, w, ids):
    """Logits at every position in f64, one dense mask; K and V as the caches hold them."""
    from ttsxabe_amd.gpu import rope_scaling
    w = {k: torch.from_numpy(v).double() for k, v in w.items()}
    n, hd = len(ids), cfg.head_dim
    norm = lambda x, g: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg.eps) * g  # noqa: E731
    rot = cfg.rope_dim or hd
    div, theta, m = rope_scaling(rot, cfg.theta, *(cfg.rope_scaling or ("none",)), device="cpu")
    turn = lambda x: ref.rotate(x, torch.arange(n), rot, theta, div, m, cfg.rope_interleaved)  # noqa: E731
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    seen = (j <= i) & ((j > i - cfg.window) | (j < cfg.shared)) if cfg.window else j <= i
    h = w["embed"][torch.tensor(ids)]
    for l in range(cfg.layers):
        x = norm(h, w[f"{l}.attn_norm"])
        q = turn((x @ w[f"{l}.wq"].T).view(n, cfg.heads, hd))
        k = turn((x @ w[f"{l}.wk"].T).view(n, cfg.kv_heads, hd)).half().double()
        v = (x @ w[f"{l}.wv"].T).view(n, cfg.kv_heads, hd).half().double()
        slopes = None if cfg.slopes is None else torch.tensor(cfg.slopes)
        ctx, _ = ref.attend(q, k.transpose(0, 1), v.transpose(0, 1), seen, torch.arange(n), hd ** -0.5, cfg.softcap, slopes)
        h = h + ctx.reshape(n, -1) @ w[f"{l}.wo"].T
        x = norm(h, w[f"{l}.ffn_norm"])
        h = h + (torch.nn.functional.silu(x @ w[f"{l}.wg"].T) * (x @ w[f"{l}.wu"].T)) @ w[f"{l}.wd"].T
    return (norm(h, w["norm"]) @ w["lm_head"].T).numpy()


@pytest.mark.parametrize("cfg", [
    Config(softcap=5.0, rope_dim=32, rope_interleaved=True, rope_scaling=("yarn", 4.0, 64)),
    Config(window=24, shared=3, rope_scaling=("linear", 2.0, 64)),
    Config(window=24, slopes=tuple(2.0 ** -(h + 1) for h in range(8)), rope_scaling=("ntk", 4.0, 64)),
    Config(softcap=3.0, window=200, shared=8, slopes=(0.5, 0.25, 0.1, 0.0), head_dim=128, heads=4, kv_heads=4, hidden=256),
], ids=["capped", "windowed", "biased", "all"])
def test_scores_and_positions_through_the_stack(gpu, cfg):
    from ttsxabe_amd.stack import LlamaBatch
    w = random_weights(cfg, SEED + 3)
    dev = LlamaBatch(gpu, cfg, w, slots=3, cap=128)
    texts, cuts = prompts_of(cfg, [90, 37, 15]), [80, 30, 8]
    want = [dense(cfg, w, t) for t in texts]
    got = dev.prefill([t[:c] for t, c in zip(texts, cuts)], [0, 2, 1]).cpu()
    for turn in range(7):
        for g, x, c in zip(got, want, cuts):
            near(g, x[c + turn - 1], turn)
        got = dev.step([t[c + turn] for t, c in zip(texts, cuts)], [0, 2, 1]).cpu()
    # A prompt into a slot that held another begins it anew.
    near(dev.prefill([texts[2]], [0]).cpu()[0], want[2][-1], "again")


def test_refusals(gpu):
    from ttsxabe_amd.gpu import CacheOverrun, InvalidArgument
    from ttsxabe_amd.stack import LlamaBatch
    cfg = StackConfig(layers=1)
    dev = LlamaBatch(gpu, cfg, random_weights(cfg, 1), slots=2, cap=32)
    for prompts, slots in (([[1]], [2]), ([[1]], [-1]), ([[1], [2]], [0, 0]), ([[1]], [0, 1]), ([], []), ([[]], [0])):
        with pytest.raises(InvalidArgument):
            dev.prefill(prompts, slots)
    with pytest.raises(CacheOverrun):
        dev.prefill([[1] * 33], [0])
    assert dev.length == [0, 0]
    dev.prefill([[1] * 31], [1])
    dev.step([3], [1])
    with pytest.raises(CacheOverrun):
        dev.step([3], [1])
    with pytest.raises(InvalidArgument):
        dev.step([3, 4], [1])
    assert dev.length == [0, 32]
