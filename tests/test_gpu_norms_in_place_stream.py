"""The C entry with the new stream in the place of the old one (or of the rows themselves): the results of a call with a tensor of its own."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,H", [(12, 1024), (12, 1001), (3000, 512)])
@pytest.mark.parametrize("place", ["residual", "x"])
def test_same_results(T, H, place):
    from liquidgemm_b200 import norms
    from liquidgemm_b200._lib import lib
    gen = torch.Generator(device="cuda").manual_seed(H)
    x, r, w = (torch.randn(*s, device="cuda", generator=gen) for s in ((T, H), (T, H), (H,)))
    r[2], r[3], x[3] = 3e38, 0.0, 0.0
    r[4] *= 1e-30
    x[4] *= 1e-30
    x[5] *= 1e30
    for post in (None, w):
        z, h = norms.block_norm(x, w, residual=r, post_weight=post, eps=0.0)
        got_z, got_x, got_r = torch.empty_like(x), x.clone(), r.clone()
        into = got_r if place == "residual" else got_x
        code = lib.lq_block_norm(got_x.data_ptr(), 2, 0, H, got_r.data_ptr(), 2, 0, H, None, 2, 0, 0, 0, w.data_ptr(), 2,
                                 None if post is None else post.data_ptr(), 2, got_z.data_ptr(), None, None, into.data_ptr(), T, T, H, 0.0, 1.0, 1.0,
                                 0.0, torch.cuda.current_stream().cuda_stream)
        assert code == 0
        assert torch.equal(into, h) and torch.equal(got_z, z)
