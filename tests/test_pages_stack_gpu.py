"""The operators over pages together, as they are used: `LlamaPages` begins
sequences, begins others behind them, steps all of them over shared and
selected pages and gives pages back. Logits against the CPU restatement of the
plain stack and the dense 64-bit one, by the rule of test_batch_gpu.py."""
from dataclasses import dataclass

import numpy as np
import pytest
import torch

import ranges_ref as ref
from oracle.stack import CpuStack, StackConfig, random_weights
from test_batch_gpu import Config, dense, near, prompts_of
from tests.configs import SEED

pytestmark = pytest.mark.gpu


@dataclass(frozen=True)
class Selecting(StackConfig):
    select: tuple = (4, 1, 1)


def test_sequences_behind_a_document(gpu):
    """A document, three questions behind it in one pass (its last page not full), one behind one of those, and an
    unrelated prompt: all stepped together, in different orders, against a CPU stack each."""
    from ttsxabe_amd.stack import LlamaPages
    cfg = StackConfig()
    w = random_weights(cfg, SEED)
    dev = LlamaPages(gpu, cfg, w, slots=7, cap=400, pages=60, page=32)
    doc, *rest = prompts_of(cfg, [150, 9, 1, 40, 17, 70])
    near(dev.prefill([doc], [3]).cpu()[0], CpuStack(cfg, w).forward(doc), "document")
    full = {0: doc + rest[0], 6: doc + rest[1], 2: doc + rest[2]}
    got = dev.prefill(rest[:3], [0, 6, 2], behind=3).cpu().numpy()
    cpus = {s: CpuStack(cfg, w) for s in full}
    want = {s: cpus[s].forward(t) for s, t in full.items()}
    for g, s in zip(got, [0, 6, 2]):
        near(g, want[s], ("behind", s))
    assert all(dev.own[s][:4] == dev.own[3][:4] and dev.own[s][4] != dev.own[3][4] for s in full)
    cpus[5], cpus[1] = CpuStack(cfg, w), CpuStack(cfg, w)
    want[5] = cpus[5].forward(full[2] + rest[3])
    near(dev.prefill([rest[3]], [5], behind=2).cpu()[0], want[5], "behind a question")
    want[1] = cpus[1].forward(rest[4])
    near(dev.prefill([rest[4]], [1]).cpu()[0], want[1], "unrelated")
    order, starts, prefix = dev._groups([5, 1, 0, 6, 2])
    assert sum(p > 0 for p in prefix) == 1 and max(prefix) == 128
    for turn in range(6):
        slots = [[5, 1, 0, 6, 2], [2, 0], [6, 5, 2, 1, 0]][turn % 3]
        ids = [int(want[s].argmax()) for s in slots]
        for s, t in zip(slots, ids):
            want[s] = cpus[s].forward([t])
        got = dev.step(ids, slots).cpu().numpy()
        for g, s in zip(got, slots):
            near(g, want[s], (turn, s))
    assert [dev.length[s] for s in (0, 6, 2, 5, 1)] == [cpus[s].past for s in (0, 6, 2, 5, 1)]
    # The document ends: what the others hold of it stays.
    dev.free([3])
    t = int(want[0].argmax())
    near(dev.step([t], [0]).cpu()[0], cpus[0].forward([t]), "after the document")
    dev.free([0, 6, 2, 5, 1])
    assert sorted(dev.spare) == list(range(60)) and not any(dev.held) and dev.length == [0] * 7


@pytest.mark.parametrize("cfg", [
    Config(softcap=5.0, rope_dim=32, rope_interleaved=True, rope_scaling=("yarn", 4.0, 64)),
    Config(window=40, shared=3, rope_scaling=("linear", 2.0, 64)),
    Config(softcap=3.0, window=70, shared=8, slopes=(0.5, 0.25, 0.1, 0.0), head_dim=128, heads=4, kv_heads=4, hidden=256),
], ids=["capped", "windowed", "all"])
def test_scores_and_positions_behind_a_document(gpu, cfg):
    from ttsxabe_amd.stack import LlamaPages
    w = random_weights(cfg, SEED + 3)
    dev = LlamaPages(gpu, cfg, w, slots=4, cap=160, pages=24, page=32)
    doc, *rest = prompts_of(cfg, [70, 40, 33, 9])
    texts, cuts = [doc + r for r in rest], [70 + 30, 70 + 20, 70 + 2]
    want = [dense(cfg, w, t) for t in texts]
    near(dev.prefill([doc], [1]).cpu()[0], want[0][69], "document")
    got = dev.prefill([t[70:c] for t, c in zip(texts, cuts)], [0, 2, 3], behind=1).cpu()
    for turn in range(7):
        for g, x, c in zip(got, want, cuts):
            near(g, x[c + turn - 1], turn)
        got = dev.step([t[c + turn] for t, c in zip(texts, cuts)], [0, 2, 3]).cpu()


def sparse(cfg, w, ids, page, lead):
    """Logits of the last token in f64 where the rows from `lead` on attend selected pages."""
    count, first, last = cfg.select
    w = {k: torch.from_numpy(v).double() for k, v in w.items()}
    n, hd, kv = len(ids), cfg.head_dim, cfg.kv_heads
    norm = lambda x, g: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg.eps) * g  # noqa: E731
    h = w["embed"][torch.tensor(ids)]
    for l in range(cfg.layers):
        x = norm(h, w[f"{l}.attn_norm"])
        q = ref.rotate((x @ w[f"{l}.wq"].T).view(n, cfg.heads, hd), torch.arange(n), hd, cfg.theta)
        k = ref.rotate((x @ w[f"{l}.wk"].T).view(n, kv, hd), torch.arange(n), hd, cfg.theta).half().double()
        v = (x @ w[f"{l}.wv"].T).view(n, kv, hd).half().double()
        ctx = torch.zeros(n, cfg.heads, hd, dtype=torch.float64)
        for r in range(n):
            live = (r + page) // page
            for g in range(kv):
                hs = slice(g * (cfg.heads // kv), (g + 1) * (cfg.heads // kv))
                keep = torch.ones(r + 1, dtype=torch.bool)
                if r >= lead and live > count:
                    score = torch.full((live,), torch.inf, dtype=torch.float64)
                    for p in range(first, live - last):
                        b = k[p * page:(p + 1) * page, g]
                        score[p] = (q[r, hs].clamp(min=0) @ b.amax(0) + q[r, hs].clamp(max=0) @ b.amin(0)).max()
                    best = score.sort(descending=True, stable=True).indices[:count]
                    keep = torch.isin(torch.arange(r + 1) // page, best)
                p = torch.softmax((q[r, hs] @ k[:r + 1, g].T * hd ** -0.5).masked_fill(~keep, -torch.inf), -1)
                ctx[r, hs] = p @ v[:r + 1, g]
        h = h + ctx.reshape(n, -1) @ w[f"{l}.wo"].T
        x = norm(h, w[f"{l}.ffn_norm"])
        h = h + (torch.nn.functional.silu(x @ w[f"{l}.wg"].T) * (x @ w[f"{l}.wu"].T)) @ w[f"{l}.wd"].T
    return (norm(h, w["norm"]) @ w["lm_head"].T)[-1].numpy()


def test_selected_pages_through_the_stack(gpu):
    """Steps over 4 of up to 10 pages, through one layer (behind a first one's rounding a second may choose otherwise
    than f64 does)."""
    from ttsxabe_amd.stack import LlamaBatch, LlamaPages, LlamaStack
    cfg = Selecting(layers=1)
    w = random_weights(cfg, SEED + 5)
    dev = LlamaPages(gpu, cfg, w, slots=3, cap=330, pages=40, page=32)
    texts = prompts_of(cfg, [305, 100, 200])
    dev.prefill([t[:-3] for t in texts], [2, 0, 1])
    for i in range(3):
        got = dev.step([t[len(t) - 3 + i] for t in texts], [2, 0, 1]).cpu().numpy()
    for g, t in zip(got, texts):
        near(g, sparse(cfg, w, t, 32, len(t) - 3), len(t))
    for other in (lambda: LlamaBatch(gpu, cfg, w, 1, 64), lambda: LlamaStack(gpu, cfg, w)):
        with pytest.raises(ValueError):
            other()
    with pytest.raises(ValueError):
        LlamaPages(gpu, dataclass(frozen=True)(type("C", (Selecting,), {"window": 9}))(), w, 1, 64, 4, 32)


def test_refusals(gpu):
    from ttsxabe_amd.gpu import CacheOverrun, InvalidArgument
    from ttsxabe_amd.stack import LlamaPages
    cfg = StackConfig(layers=1)
    dev = LlamaPages(gpu, cfg, random_weights(cfg, 1), slots=3, cap=96, pages=4, page=32)
    for prompts, slots in (([[1]], [3]), ([[1]], [-1]), ([[1], [2]], [0, 0]), ([[1]], [0, 1]), ([], []), ([[]], [0]),
                           ([[512]], [0]), ([[-1]], [0])):
        with pytest.raises(InvalidArgument):
            dev.prefill(prompts, slots)
    for behind in (0, 1, 3, -1):  # itself, none begun, no slots
        with pytest.raises(InvalidArgument):
            dev.prefill([[1]], [0], behind=behind)
    with pytest.raises(CacheOverrun):
        dev.prefill([[1] * 97], [0])
    with pytest.raises(InvalidArgument):
        dev.step([1], [0])
    dev.prefill([[1] * 64], [0])
    with pytest.raises(CacheOverrun):  # five pages of four
        dev.prefill([[1] * 65], [1])
    assert dev.length == [64, 0, 0] and len(dev.spare) == 2 and not dev.own[1]
    dev.prefill([[2] * 40], [1], behind=None)
    with pytest.raises(CacheOverrun):  # a page for its next token
        dev.step([3], [0])
    assert dev.length == [64, 40, 0]
    dev.free([1])
    dev.prefill([[3] * 96], [0])  # in the pages that it had and the other left
    assert dev.length == [96, 0, 0] and len(dev.spare) == 1
