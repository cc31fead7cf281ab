"""What LlamaPages does on the host about who holds which page, without a device."""
import random

import pytest
import torch

from ttsxabe_amd.gpu import CacheOverrun
from ttsxabe_amd.stack import LlamaPages


class Pages(list):
    """A sequence's pages; counts how many were looked at."""
    looked = 0

    def __iter__(self):
        Pages.looked += len(self)
        return super().__iter__()

    def __contains__(self, p):
        Pages.looked += len(self)
        return super().__contains__(p)


def held(own, pages, page=32, cap=10**6):
    x = LlamaPages.__new__(LlamaPages)
    x.page, x.cap, x.slots, x.w = page, cap, len(own), {"embed": [0] * 10}
    x.own = [Pages(s) for s in own]
    x.held = [sum(p in s for s in own) for p in range(pages)]
    x.spare = [p for p in range(pages) if not x.held[p]]
    x.length = [page * len(s) for s in own]
    return x


@pytest.mark.parametrize("seed", range(5))
def test_pages_that_new_prompts_find(seed):
    """A prompt that is one page too long is refused with the pages that its slot's end would leave, those that others
    hold not among them; each page held is looked at a few times at most."""
    r = random.Random(seed)
    pages, own, at = 700, [], 0
    for t in range(8):
        lead = r.choice(own)[:r.randint(0, 40)] if own and r.random() < 0.7 else []
        n = r.randint(0, 60)
        own.append(lead + list(range(at, at + n)))
        at += n
    for k in (1, 3, 8):
        slots = r.sample(range(8), k)
        x = held(own, pages)
        others = {p for t in range(8) if t not in slots for p in own[t]}
        room = pages - len(others)
        Pages.looked = 0
        with pytest.raises(CacheOverrun) as e:
            x.prefill([[1] * (32 * (room + 2 - k) if t == 0 else 1) for t in range(k)], slots)
        assert e.value.fields == (room + 1, room)
        assert Pages.looked <= 2 * sum(map(len, own))
        assert x.own == own and x.length == [32 * len(s) for s in own]


@pytest.mark.parametrize("behind", [None, 3])
def test_prompts_that_fail(behind):
    """A pass that ends in an error begins nothing: its slots are empty, their pages are back, others are as they were."""
    x = held([[0, 1], [2], [], [3, 4, 5]], 20)
    x.length[3] = 70  # its third page is not full

    class Device:
        device = "cpu"

        def __getattr__(self, name):
            raise MemoryError(name)

    x.g, x.cache, x.window, x.shared = Device(), [], 0, 0
    x.table = torch.full((4, 10), -1, dtype=torch.int32)
    x.cfg = type("Cfg", (), {"heads": 4, "head_dim": 64, "kv_heads": 4})
    x.cache = [type("Cache", (), {"pages": 20, "data": torch.zeros(20, 8)})]
    with pytest.raises(MemoryError):
        x.prefill([[1] * 40, [2] * 5], [0, 2], behind=behind)
    assert x.length == [0, 32, 0, 70] and [list(s) for s in x.own] == [[], [2], [], [3, 4, 5]]
    assert sorted(x.spare) == [0, 1] + list(range(6, 20)) and [p for p in range(20) if x.held[p]] == [2, 3, 4, 5]
    assert all(x.held[p] == 1 for p in (2, 3, 4, 5))
