"""The clip over numbers of tensors around a launch's, empty ones among them and behind them."""
import pytest

from sushi_amd import exl3
from tests.test_gpu_clip import BF16, F16, F32, _exact, _grads, _matches

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [159, 160, 161, 319, 320, 321])
@pytest.mark.parametrize("empty", ["none", "every third", "the last ones", "the first ones"])
def test_tensors_around_a_launch(dev, count, empty):
    sizes = [(1, 8191, 8192, 8193, 77, 20000)[i % 6] for i in range(count)]
    if empty == "every third":
        sizes = [n for s in sizes for n in ((s, s, 0) if s == 77 else (s,))][:count]
    elif empty == "the last ones":
        sizes += [0] * 170
    elif empty == "the first ones":
        sizes = [0] * 170 + sizes
    grads = _grads(dev, sizes, [F32, BF16, F16])
    norm, _ = _exact(grads, 1.0)
    mine = [t.clone() for t in grads]
    _matches(grads, mine, exl3.clip_grad_norm(mine, norm * 0.3), norm * 0.3)
