"""Forms of the 4-bit KV cache kernels that only many rows, heads or sequences reach: four heads per lane
group in append and read-back, against one head per group (which the other tests compare with the
definition); read-back into fp16; whole items in turn in the attention."""
import numpy as np
import pytest

import vsl
from test_kv_q4_gpu import Cache, check_append, check_attend, dev, rope_tables

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def lanes_of_few_heads():
    """Lanes up to which a lane group takes one head."""
    return torch.cuda.get_device_properties(0).multi_processor_count * 2048


@pytest.mark.parametrize("kvdt", [vsl.Q4_0, vsl.F16, vsl.F32])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (5, 3, 64), (1, 1, 64), (32, 8, 128), (7, 1, 128), (3, 3, 128)])
@pytest.mark.parametrize("style", [vsl.ROPE_ADJACENT, vsl.ROPE_HALVES])
def test_four_heads_per_group_store_what_one_does(kvdt, nh, nkv, hd, style):
    """Bit for bit, with head counts that are multiples of four and not; the codes of a token do not depend on
    the rows it arrives with."""
    rng = np.random.default_rng(nh + nkv + hd + style)
    heads, page = nh + 2 * nkv, 64
    n = lanes_of_few_heads() // (heads * (hd // 4)) + 5
    piece = n // 2
    x = torch.randn(n, heads * hd, device="cuda")
    wq, wk = (dev((0.5 + rng.random(hd)).astype(np.float32)) for _ in range(2))
    cos, sin = (dev(a) for a in rope_tables(n, hd))
    pos = dev(rng.permutation(n).astype(np.int32))
    seq = torch.zeros_like(pos)
    table = rng.permutation(-(-n // page) + 2)[:-(-n // page)].reshape(1, -1)
    many, few = (Cache(kvdt, table.size + 2, nkv, hd, page, table) for _ in range(2))
    q = many.append(x, nh, wq, wk, seq, pos, cos, sin, style)
    for a in range(0, n, piece):
        b = min(a + piece, n)
        assert torch.equal(few.append(x[a:b], nh, wq, wk, seq[a:b], pos[a:b], cos, sin, style), q[a:b])
    assert torch.equal(many.k, few.k) and torch.equal(many.v, few.v)
    assert many.status.item() == 0 and few.status.item() == 0


def test_append_of_many_rows_of_few_heads():
    check_append(vsl.Q4_0, 5, 3, 64, 64, 3, [900, 700, 300], vsl.ROPE_HALVES, True, True, seed=61)
    check_append(vsl.F16, 5, 3, 64, 128, 2, [1000, 900], vsl.ROPE_ADJACENT, True, True, seed=62)


@pytest.mark.parametrize("kvdt", [vsl.Q4_0, vsl.F16, vsl.F32])
@pytest.mark.parametrize("nkv,hd", [(8, 128), (3, 64), (1, 64), (5, 128)])
def test_read_back_of_many_rows_and_into_fp16(kvdt, nkv, hd):
    rng = np.random.default_rng(nkv + hd)
    page, nh = 64, 1
    n = lanes_of_few_heads() // (2 * nkv * (8 if kvdt == vsl.Q4_0 else hd // 4)) + 3
    held = -(-n // page)
    c = Cache(kvdt, held + 1, nkv, hd, page, rng.permutation(held + 1)[:held].reshape(1, -1))
    pos = dev(rng.permutation(n).astype(np.int32))
    seq = torch.zeros_like(pos)
    c.append(torch.randn(n, (nh + 2 * nkv) * hd, device="cuda"), nh, None, None, seq, pos, None, None, 0)
    pos[::7] = -1  # padding in between
    for out in (torch.float32, torch.float16):
        whole = c.read(seq, pos, out)
        piece = n // 2
        for a in range(0, n, piece):
            part = c.read(seq[a:a + piece].contiguous(), pos[a:a + piece].contiguous(), out)
            assert all(torch.equal(p, w[a:a + piece]) for p, w in zip(part, whole))
        assert all((w[::7] == 0).all() for w in whole)
        if out == torch.float32:
            wide = whole
        else:
            assert all(torch.equal(w, f.half()) for w, f in zip(whole, wide))
    assert c.status.item() == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv,rows", [(8, 8, 1), (16, 8, 3), (4, 4, 20)])
def test_more_items_than_warps(hd, nh, nkv, rows):
    """Every warp takes whole items in turn, some one more than others; empty sequences, lengths around the
    stage, some longer ones."""
    warps = torch.cuda.get_device_properties(0).multi_processor_count * 12
    tiles = -(-rows * (nh // nkv) // 8)
    B = warps // (nkv * tiles) + 9
    assert B <= 1024 and B * nkv * tiles > warps
    check_attend(hd + nh + rows, nh, nkv, hd, [(37 * i) % 170 if i % 50 else 400 for i in range(B)], rows, 64)
    check_attend(hd + rows, nh, nkv, hd, [(53 * i) % 300 for i in range(B)], rows, 64, mask=(100, 40, 4, 128))


def test_as_many_items_as_warps():
    """One item per warp, and one fewer and one more."""
    warps = torch.cuda.get_device_properties(0).multi_processor_count * 12
    for B in (warps // 4 - 1, warps // 4, warps // 4 + 1):
        check_attend(B, 4, 4, 64, [1 + (41 * i) % 100 for i in range(B)], 1, 64)
