"""examples/moe_layer.py: the products together, as a layer is trained and served."""
import importlib.util
import pathlib

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = pathlib.Path(__file__).resolve().parent.parent / "examples" / "moe_layer.py"


@pytest.mark.parametrize("tokens,width,hidden,experts", [(1024, 256, 512, 8), (257, 130, 264, 5)])
def test_the_layer_learns_and_serves_in_8_bits(cuda, tokens, width, hidden, experts):
    spec = importlib.util.spec_from_file_location("moe_layer", EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, deviation = example.main(tokens, width, hidden, experts, steps=25, quiet=True)
    assert losses[-1] < 0.8 * losses[0]
    assert all(loss == loss for loss in losses)
    # e4m3 keeps 4 significant bits: 2^-4 at most for a value, about 2.6 % in
    # norm for each of the two products' four operands.
    assert deviation < 0.08
