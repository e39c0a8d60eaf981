"""decode.PagedDecodeStep behind shared prefixes whose sequences end in any order.  Reference and tolerance as in
test_gpu_shared_serving.py."""
from __future__ import annotations

import pytest

from qorvix_amd import decode
from test_gpu_serving import _model, _near
from test_gpu_shared_serving import HostShared, _both

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_pages", [12, 1 << 18])
@pytest.mark.parametrize("gone", [[0], [0, 1], [0, 2], [1]])
@pytest.mark.parametrize("replay", [False, True])
def test_samples_of_a_prompt_end_in_any_order(cuda, gone, replay, max_pages):
    """Four samples of a prompt in one group; some are released, the first one too, and the others go on as they were, also
    where the pages that went back hold other tokens by then.  The second width reads the prefix in a launch of its own."""
    torch = cuda
    torch.manual_seed(3)
    m, page = 4, 4
    step = decode.PagedDecodeStep(_model(torch, layers=1), m, heads=8, kv_heads=2, n_pages=24, max_pages=max_pages, page_size=page,
                                  shared_groups=1)
    host = HostShared(torch, step, torch.float16)
    _both(torch, step, host, 10)
    step.fork([0] * 3, [1, 2, 3])
    host.fork([0] * 3, [1, 2, 3])
    step.shared[0] = 10 // page * page
    _both(torch, step, host, 3)
    if replay:
        step.capture()
    step.release(gone)
    host.empty(gone)
    stay = [b for b in range(m) if b not in gone]
    for _ in range(6):  # fewer than the shared tokens
        x = torch.randn((m, 512), device="cuda")
        want_x, want = host.run(x)
        step.x.copy_(x)
        if replay:
            step.replay()
        else:
            step.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert step.taken.tolist()[1] == 0 and step.lens.tolist() == host.t
        _near(step.x[stay], want_x[stay], 8e-3)
        _near(step.logits[stay], want[stay], 8e-3)
