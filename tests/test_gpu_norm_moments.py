"""Group norm of data whose first values are not like the rest (a corner that
was never touched, one outlier): the statistics are as good as for typical
data, in each of the kernel's three forms.  Tolerances are those of
test_gpu_ops.check_norm, derived there for sums of centred values."""
import pytest
import torch

from ssla_rt_b200 import ops
from test_gpu_ops import DT, check_norm, rand

pytestmark = pytest.mark.gpu

# (samples, positions, channels, groups): slabs in registers, in a cluster's shared memory (wide and single-value
# vectors), and larger ones; one larger slab whose threads each walk many positions
FORMS = [(2, 40, 24, 2), (2, 5120, 96, 8), (3, 5001, 33, 11), (1, 120001, 96, 8), (2, 70000, 15, 1), (1, 2000003, 8, 1)]
DATA = [(500.0, 1.0, 500.0), (10.0, 0.1, 0.0), (500.0, 1.0, 0.0), (0.0, 1.0, 1000.0), (0.0, 1.0, 10000.0), (100.0, 1.0, 0.0)]


def data(n, p, c, mean, std, first, rows, dtype):
    x = (rand(p + c, n, p, c) * std + mean)
    x[:, :rows] = first
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("mean,std,first", DATA)
def test_first_position_is_not_typical(dtype, form, mean, std, first):
    n, p, c, g = form
    x = data(n, p, c, mean, std, first, 1, DT[dtype])
    check_norm(x, g, None, None, "none", ops.group_norm(x, g, activation="none"))


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("where", [0, 1, -1])
def test_one_outlier(form, where):
    n, p, c, g = form
    x = data(n, p, c, 3.0, 1.0, 3.0, 0, torch.float32)
    x[:, where, ::c // g] = -20000.0
    w, b = 1 + 0.2 * rand(2, c), 0.1 * rand(3, c)
    check_norm(x, g, w, b, "silu", ops.group_norm(x, g, w, b))


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_a_zero_border(form):
    """A tenth of the positions at zero, then values far from it, with little spread."""
    n, p, c, g = form
    x = data(n, p, c, 40.0, 0.5, 0.0, max(1, p // 10), torch.float32)
    check_norm(x, g, None, None, "none", ops.group_norm(x, g, activation="none"))


def test_a_drift_over_the_positions():
    """Values that move by many times their spread from the first position to the last."""
    x = rand(5, 1, 200000, 16) * 0.01 + torch.linspace(0, 100, 200000, device="cuda")[None, :, None]
    check_norm(x, 2, None, None, "none", ops.group_norm(x, 2, activation="none"))
