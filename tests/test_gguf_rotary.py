"""A GGUF's rotary metadata (`llama.rope.*`) in a Llama's configuration."""
import math

import pytest

from oracle.stack import StackConfig, random_weights
from test_gguf import llama_gguf
from ttsxabe_amd import gguf
from ttsxabe_amd.llama_gguf import LlamaGgufError, config_from_gguf, load_llama_gguf

CFG = StackConfig(vocab=64, hidden=128, heads=4, kv_heads=2, head_dim=32, ffn=256, layers=1)


def with_metadata(path, more):
    """A Llama's file with `more` metadata."""
    llama_gguf(path, CFG, random_weights(CFG, 3))
    f = gguf.GgufFile.open(path)
    meta = {k: (f._tags[k], v) for k, v in f.metadata.items()}
    tensors = [(t.name, t.type_name, t.dims, f.tensor_bytes(t.name).tobytes()) for t in f.tensors]
    gguf.write_gguf(path, {**meta, **more}, tensors)
    return gguf.GgufFile.open(path)


def scaling(kind, factor=None, original=None, context=None):
    m = {"llama.rope.scaling.type": (gguf.STRING, kind)}
    if factor is not None:
        m["llama.rope.scaling.factor"] = (gguf.F32, factor)
    if original is not None:
        m["llama.rope.scaling.original_context_length"] = (gguf.U32, original)
    if context is not None:
        m["llama.context_length"] = (gguf.U32, context)
    return m


@pytest.mark.parametrize("kind", ["linear", "yarn"])
def test_scaled_positions(tmp_path, kind):
    f = with_metadata(tmp_path / "m.gguf", scaling(kind, 4.0, 4096, 16384))
    assert config_from_gguf(f).rope_scaling == (kind, 4.0, 4096)
    for interleaved in (False, True):
        assert load_llama_gguf(f, interleaved)[0].rope_scaling == (kind, 4.0, 4096)


def test_the_original_context_is_the_whole_one_where_no_other_is_named(tmp_path):
    from ttsxabe_amd.gpu import rope_scaling
    c = config_from_gguf(with_metadata(tmp_path / "m.gguf", scaling("yarn", 4.0, None, 2048)))
    assert c.rope_scaling == ("yarn", 4.0, 2048)
    div, _, m = rope_scaling(c.head_dim, c.theta, *c.rope_scaling, device="cpu")
    turns = [2048 / (2 * math.pi) * c.theta ** (-i / 16) for i in range(16)]
    assert [float(d) == 4.0 for d in div] == [t <= 1.0 for t in turns]
    assert math.isclose(m, 1.0 + 0.1 * math.log(4.0))


def test_yarn_without_any_context_is_refused(tmp_path):
    f = with_metadata(tmp_path / "m.gguf", scaling("yarn", 4.0))
    with pytest.raises(LlamaGgufError, match="original_context_length"):
        config_from_gguf(f)


def test_linear_positions_need_no_context(tmp_path):
    c = config_from_gguf(with_metadata(tmp_path / "m.gguf", scaling("linear", 2.0)))
    assert c.rope_scaling[:2] == ("linear", 2.0)


@pytest.mark.parametrize("more", [{}, scaling("none", 4.0, 4096), scaling("linear"), scaling("yarn", None, 4096)])
def test_positions_are_unscaled(tmp_path, more):
    assert config_from_gguf(with_metadata(tmp_path / "m.gguf", more)).rope_scaling is None


def test_rotated_dims(tmp_path):
    """The count is for the file's own order of dims; unpermuted (whole) heads are rotated whole."""
    f = with_metadata(tmp_path / "m.gguf", {"llama.rope.dimension_count": (gguf.U32, 16)})
    assert config_from_gguf(f).rope_dim == 16
    c, _ = load_llama_gguf(f, interleaved=True)
    assert c.rope_dim == 16 and c.rope_interleaved
    c, _ = load_llama_gguf(f)
    assert c.rope_dim == 0 and not c.rope_interleaved


@pytest.mark.parametrize("more,what", [
    (scaling("longrope", 4.0, 4096), "longrope"), (scaling("other"), "other"),
    ({**scaling("yarn", 4.0, 4096), "llama.rope.scaling.attn_factor": (gguf.F32, 0.75)}, "attn_factor"),
], ids=["longrope", "other", "attn_factor"])
def test_scalings_that_are_not_computed_are_refused(tmp_path, more, what):
    f = with_metadata(tmp_path / "m.gguf", more)
    with pytest.raises(LlamaGgufError, match=what):
        config_from_gguf(f)


def test_a_factor_of_one_multiplies_nothing(tmp_path):
    m = {**scaling("linear", 4.0, 4096), "llama.rope.scaling.attn_factor": (gguf.F32, 1.0)}
    assert config_from_gguf(with_metadata(tmp_path / "m.gguf", m)).rope_scaling == ("linear", 4.0, 4096)
