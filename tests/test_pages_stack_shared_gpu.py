"""LlamaPages where what sequences share is long enough that a step has tiles of it: a document of more than 640
positions, more sequences behind it than a tile takes rows, against the dense 64-bit stack. The plans that the
stack makes are looked at for such tiles (flag 2 of an item)."""
import pytest
import torch

from oracle.stack import StackConfig, random_weights
from test_batch_gpu import Config, dense, near, prompts_of
from test_paged_shared_gpu import tiles
from tests.configs import SEED

pytestmark = pytest.mark.gpu


class Watched:
    """The device with its plans held on to."""

    def __init__(self, gpu):
        self.gpu, self.plans = gpu, []

    def __getattr__(self, name):
        return getattr(self.gpu, name)

    def page_plan(self, *a, **k):
        self.plans.append(self.gpu.page_plan(*a, **k))
        return self.plans[-1]

    def shared(self):
        """(first row, rows) of the last plan's shared tiles."""
        return set(tiles(self.plans[-1], self.plans[-1].tk.numel()))


@pytest.mark.parametrize("cfg,rows", [
    (Config(), 8),
    (Config(slopes=tuple(2.0 ** -i for i in range(1, 9))), 8),
    (Config(heads=12, kv_heads=1, slopes=tuple(2.0 ** -(1 + i / 2) for i in range(12)), softcap=20.0), 2),
    (Config(heads=6, slopes=(0.3, 0.2, 0.1, 0.05, 0.025, 0.0125), window=500, shared=16), 10),
], ids=["plain", "biased", "twelve", "windowed"])
def test_one_more_sequence_than_a_tile(gpu, cfg, rows):
    """A document, a question each for one sequence more than a tile takes rows of, begun in one pass of which the last
    question is one row more than its tiles, then steps of all and of some."""
    from ttsxabe_amd.stack import LlamaPages
    w = random_weights(cfg, SEED + 3)
    n, lead, long = rows + 1, 675, 672
    dev = LlamaPages(Watched(gpu), cfg, w, slots=n + 1, cap=740, pages=21 + 4 * (n + 1), page=32)
    doc, *rest = prompts_of(cfg, [lead] + [9 + t % 3 for t in range(n)])
    texts, cuts = [doc + r for r in rest], [lead + 1 + t % 2 for t in range(n)]
    # One row more than whole tiles in all, the last prompt's last.
    more = (1 - sum(c - lead for c in cuts)) % rows
    cuts[0] += min(more, 7)
    cuts[1] += more - min(more, 7)
    want = [dense(cfg, w, t) for t in texts]
    near(dev.prefill([doc], [n]).cpu()[0], want[0][lead - 1], "document")
    got = dev.prefill([t[lead:c] for t, c in zip(texts, cuts)], list(range(n)), behind=n).cpu()
    total = sum(c - lead for c in cuts)
    assert total % rows == 1 and (total - 1, 1) in dev.g.shared()
    for turn in range(2):
        for t, (g, x, c) in enumerate(zip(got, want, cuts)):
            near(g, x[c + turn - 1], (turn, t))
        got = dev.step([t[c + turn] for t, c in zip(texts, cuts)], list(range(n))).cpu()
        assert dev.g.shared() == {(0, rows), (rows, 1)}
    assert max(dev._groups(list(range(n)))[2]) == long
    some = [n - 1, 0, n // 2]
    for g, t in zip(got, range(n)):
        near(g, want[t][cuts[t] + 1], ("all", t))
    got = dev.step([texts[t][cuts[t] + 2] for t in some], some).cpu()
    for g, t in zip(got, some):
        near(g, want[t][cuts[t] + 2], ("some", t))
