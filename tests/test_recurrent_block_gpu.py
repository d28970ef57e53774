"""The example that runs the norm, the 8-bit product and the recurrence together with the
GDN-2 mixer: it learns, and its 8-bit serving follows the float32 stack.

8 bits: a row's step is max / 127; the four roundings in a block (norm's output, mixer's
output, two weights) are uniform within a step, each about 0.3 of a step of a row whose
largest value is about 3.5 times its rms: 0.8% each, 1.6% a block, and bfloat16 values
between the kernels 0.2% each; over two blocks below 5% of the output's rms.  Prompt and
single tokens against the whole sequence at once go the same way but for the mixers'
rounding (bfloat16 tiles against float32 steps), which can turn single 8-bit values:
below 2%."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_example_learns_and_serves(dev):
    path = Path(__file__).resolve().parents[1] / "examples" / "recurrent_block.py"
    spec = importlib.util.spec_from_file_location("recurrent_block", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses, off, same = mod.main()
    assert losses[-1] < 0.7 * losses[0]
    assert off < 0.05 and same < 0.02
