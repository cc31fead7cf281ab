"""What the stacks refuse before they touch a device: on a machine with no GPU."""
from dataclasses import dataclass

import pytest

from oracle.stack import StackConfig, random_weights


@dataclass(frozen=True)
class Config(StackConfig):
    rope_dim: int = 0
    rope_interleaved: bool = False
    rope_scaling: tuple | None = None
    softcap: float = 0.0
    window: int = 0
    shared: int = 0
    slopes: tuple | None = None


@pytest.mark.parametrize("extra", [
    dict(rope_interleaved=True), dict(softcap=30.0), dict(window=64), dict(slopes=(0.5,) * 8), dict(rope_dim=32),
    dict(rope_scaling=("linear", 4.0, 8192)), dict(rope_scaling=("yarn", 8.0, 4096)), dict(rope_scaling=("ntk", 2.0, 8192)),
], ids=lambda e: "-".join(e))
def test_a_plain_stack_refuses_what_it_does_not_compute(extra):
    from ttsxabe_amd.stack import LlamaStack
    cfg = Config(**extra)
    with pytest.raises(ValueError, match="LlamaBatch"):
        LlamaStack(None, cfg, random_weights(cfg, 1))


@pytest.mark.parametrize("extra", [
    {}, dict(rope_dim=64), dict(rope_scaling=("none", 4.0, 8192)), dict(rope_scaling=("linear", 1.0, 8192)), dict(shared=4),
], ids=lambda e: "-".join(e))
def test_a_plain_stack_takes_what_changes_nothing(extra):
    from ttsxabe_amd.stack import LlamaStack

    class Device:  # refusals come before the first use of the handle
        @property
        def device(self):
            raise LookupError

    cfg = Config(**extra)
    with pytest.raises(LookupError):
        LlamaStack(Device(), cfg, random_weights(cfg, 1))


@pytest.mark.parametrize("token", [64, -1, 2**31, 2**40])
def test_a_batch_refuses_a_token_that_has_no_embedding(token):
    """Before anything is launched (on a device such an index ends the process), and the sequences stay."""
    import torch

    from ttsxabe_amd.gpu import InvalidArgument
    from ttsxabe_amd.stack import LlamaBatch
    b = object.__new__(LlamaBatch)
    b.g, b.cfg, b.slots, b.cap, b.length, b.window, b.shared = None, StackConfig(vocab=64), 2, 32, [5, 0], 0, 0
    b.w = {"embed": torch.zeros(64, 4)}
    with pytest.raises(InvalidArgument):
        b.prefill([[1, 2], [3, token]], [0, 1])
    with pytest.raises(InvalidArgument):
        b.step([1, token], [0, 1])
    assert b.length == [5, 0]
