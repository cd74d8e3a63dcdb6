"""4-bit KV cache on the GPU at the ends of its ranges."""
import pytest

import vsl
from test_kv_q4_gpu import Cache, dev, rope_tables

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kvdt", [vsl.Q4_0, vsl.F16, vsl.F32])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("style", [vsl.ROPE_ADJACENT, vsl.ROPE_HALVES])
@pytest.mark.parametrize("n", [6, 3000])
def test_padding_rows_are_zero_whatever_the_norm(kvdt, hd, style, n):
    """eps 0, and norm weights and rotation factors that are not finite."""
    nh, nkv, page = 8, 2, 64
    c = Cache(kvdt, 4, nkv, hd, page, [[0, 1], [2, -1]])
    before = c.k.clone(), c.v.clone()
    x = torch.randn(n, (nh + 2 * nkv) * hd, device="cuda")
    w = torch.ones(hd, device="cuda")
    w[3] = float("inf")
    cos, sin = (dev(a) for a in rope_tables(128, hd))
    cos[0, 1] = float("nan")
    seq = torch.arange(n, device="cuda", dtype=torch.int32) % 3
    pad = torch.full_like(seq, -1)
    for norms in ((w, w), (w, None), (torch.ones_like(w), torch.ones_like(w))):
        c.status.zero_()
        q = c.append(x, nh, *norms, seq, pad, cos, sin, style, eps=0.0)
        assert (q == 0).all() and c.status.item() == 0
        q = c.append(x, nh, *norms, seq, pad + 129, cos, sin, style, eps=0.0)  # past the table
        assert (q == 0).all() and c.status.item() == -5
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1])
