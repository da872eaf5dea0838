"""More tokens than one launch of the rotation takes: the launches together cover each of them once."""
from __future__ import annotations

import pytest

from test_serving_operators_gpu import SENTINEL, _lib, _stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,heads", [(2**30 + 5, 1), (2**29 + 7, 2)])
def test_rotation_of_more_than_2_30_items(cuda, tokens, heads):
    """Pairs alone (head_dim 2, in place): one item a token and head. A quarter turn takes (a, b) to
    (-b, a), half a turn to (-a, -b), exactly; the positions alternate between the two by token."""
    import torch
    native = _lib()
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of free device memory")
    x = torch.empty(tokens * heads + 4, 2, dtype=torch.float16, device=cuda)  # the values behind must survive
    x[:, 0], x[:, 1] = 3.0, 0.5
    x[tokens * heads:] = SENTINEL
    positions = torch.empty(tokens, dtype=torch.int32, device=cuda)
    positions[0::2], positions[1::2] = 0, 1
    cos, sin = torch.tensor([[0.0], [-1.0]], device=cuda), torch.tensor([[1.0], [0.0]], device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    native.check(native.lib.ar_rotary_positions(x.data_ptr(), 2 * heads, 2, x.data_ptr(), 2 * heads, 2, positions.data_ptr(), tokens,
                                                heads, 2, 2, 0, 0, cos.data_ptr(), sin.data_ptr(), 2, status.data_ptr(), 1,
                                                _stream()))
    torch.cuda.synchronize()
    assert int(status) == 0
    even, odd = (x[:tokens * heads].view(tokens, heads, 2)[i::2] for i in (0, 1))
    for rows, want in ((even, (-0.5, 3.0)), (odd, (-3.0, -0.5))):
        for i in (0, 1):
            assert bool((rows[..., i] == want[i]).all())
    assert (x[tokens * heads:] == SENTINEL).all()
