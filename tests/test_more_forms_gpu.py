"""On a B200: forms of the sorted rows', gradients' and 8-bit rows' kernels that only longer steps or other row lengths take, against the definitions in 64 bits."""
import numpy as np
import pytest

import more_ops_common as M
import test_i8_gpu as I
import test_sort_rows_gpu as S
from c0ven_b200 import ops

pytestmark = pytest.mark.gpu
TYPES = S.TYPES


# --- the routing's gradient: warps that take one row after another ------------------------------------------------------


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T, E, n", [(19001, 64, 8), (20011, 33, 16), (38001, 200, 4), (19500, 512, 10)])
def test_route_grad_of_more_rows_than_warps(T, E, n, score, renorm, type):
    """148 * 16 CTAs of 8 warps are 18,944: warps take a second row, and a third, whatever the form. Rows of few assignments follow rows of many, so that what a
    row leaves in the columns' memory would be seen."""
    import torch

    rng = np.random.default_rng(T + n)
    l, ids = S.route_case(rng, T, E, n, type, 3.0)
    kept = torch.from_numpy(rng.random((T, n)) < np.where(np.arange(T) // 18944 % 2, 0.2, 0.9)[:, None]).cuda()
    ids = torch.where(kept, ids, -1)
    dw = rng.standard_normal((T, n)).astype(np.float32)
    dd = S.dev(dw)
    dd[~kept] = float("nan")
    out = torch.full((T + 1, E), 7.0, dtype=S.dtype(type), device="cuda")
    ops.route_logits_grad_device(l.data_ptr(), TYPES[type], T, E, n, ids.data_ptr(), dd.data_ptr(), out.data_ptr(), score=S.TYPES_OF_SCORE[score], renorm=renorm, scale=2.5)
    S.check_route_grad(S.host(out[:T]), S.host(l), ids.cpu().numpy(), dw, score, renorm, 2.5, type)
    assert (out[T] == 7.0).all()
