"""Which models take weights in 4 bits, without a GPU."""
import pytest

from burn_lm_b200 import preset
from burn_lm_b200.config import preset_names
from burn_lm_b200.model import Model, make_runtime, plan_of


def model(name, **kw):
    _, typed, plan = plan_of(preset(name))
    return Model(plan, make_runtime("bfloat16", "cpu", **kw), typed)


@pytest.mark.parametrize("name", preset_names())
def test_weights_in_4_bits_are_all_of_the_layers_or_refused(name):
    """A model either holds every matrix between its embedding and its output projection in 4 bits, or is refused with the name of a part that does not."""
    plain = model(name)
    without = {type(p).__name__ for p in plain.stream_parts + [p for layer in plain.layers for p in layer.parts()]
               if not p.four_bit and any(len(t.shape) >= 2 and min(t.shape[-2:]) >= 16 for t in p.tensor_specs())}
    if not without:
        assert model(name, weights="int4").layers
        return
    with pytest.raises(ValueError, match="weights in 4 bits: (" + "|".join(sorted(without)) + ") of (layer|the stream)"):
        model(name, weights="int4")


def test_the_models_that_take_them():
    taken = []
    for name in preset_names():
        try:
            model(name, weights="int4")
            taken.append(name)
        except ValueError:
            pass
    assert taken == [n for n in preset_names() if n.startswith(("llama3", "tiny"))]
