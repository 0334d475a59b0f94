"""CPU check of the Python layer's beam selection: a beam's score and its mark of being finished stand in the order of the
logits' rows; tensors in another order are refused before the library, which counts bytes, is called."""
import pytest

torch = pytest.importorskip("torch")

from strix_trellis import runtime  # noqa: E402
from test_fp8_scale_shapes import CTX, STREAM, Called, tensor  # noqa: E402


def select(scores, finished=None, plan=False):
    """3 prompts of 4 beams."""
    index = [tensor(3, 5, dtype=torch.int32) for _ in range(2)]
    call = runtime.BeamSelectPlan if plan else runtime.beam_select
    call(CTX, tensor(12, 50), scores, tensor(3, 5), *index, 4, finished=finished, stream=STREAM)


@pytest.mark.parametrize("plan", [False, True])
@pytest.mark.parametrize("shape", [(4, 3), (6, 2), (4, 1, 3), (4, 6)])
def test_other_orders(shape, plan):
    with pytest.raises(ValueError, match="scores and finished"):
        select(tensor(*shape), plan=plan)
    with pytest.raises(ValueError, match="scores and finished"):
        select(tensor(12), tensor(*shape, dtype=torch.int32), plan=plan)


@pytest.mark.parametrize("shape", [(12,), (3, 4), (1, 12), (12, 1), (3, 4, 1), (5,)])
def test_what_reaches_the_library(shape):
    """The documented shape, with prompts and beams apart or dimensions of one, and what is too short, which the library refuses."""
    with pytest.raises(Called):
        select(tensor(*shape))
    with pytest.raises(Called):
        select(tensor(12), tensor(*shape, dtype=torch.int32))
