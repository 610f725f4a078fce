"""Arguments of the paged operators' wrappers with too few dimensions: named, as other wrong ones are."""
import pytest
import torch

BF = torch.bfloat16


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _call():
    import lbw_amd as L
    return (L, L.paged_kv(5, 16, 2, bounds=True, device="cpu"), torch.zeros(3, 4, 128, dtype=BF), torch.zeros(3, 2, 128, dtype=BF),
            L.axis_rope(torch.zeros(8, 64), device="cpu"))


@pytest.mark.parametrize("starts", [None, _i32(2), _i32(4)])
@pytest.mark.parametrize("lens", [_i32(), _i32(1, 3), _i32(3, 1)])
def test_lens_that_are_no_vector(starts, lens):
    L, c, q, k, rope = _call()
    with pytest.raises(ValueError, match="lens must be"):
        L.paged_append_(c, q, k, k, _i32(3, 4), lens, rope, starts=starts)
    with pytest.raises(ValueError, match="lens must be"):
        L.attention_paged(q, c, _i32(3, 4), lens)
    with pytest.raises(ValueError, match="lens must be"):
        L.paged_select(q, c, _i32(3, 4), lens, 2)


@pytest.mark.parametrize("shape", [(), (5,), (5, 16), (5, 16, 2), (5, 16, 2, 128, 1)])
def test_caches_of_other_dimensions(shape):
    L, c, q, k, rope = _call()
    odd = L.PagedKV(torch.zeros(shape, dtype=BF), torch.zeros(shape, dtype=BF), c.bounds)
    with pytest.raises(ValueError):
        L.paged_append_(odd, q, k, k, _i32(3, 4), _i32(3), rope)
    with pytest.raises(ValueError):
        L.attention_paged(q, odd, _i32(3, 4), _i32(3))
    with pytest.raises(ValueError):
        L.paged_select(q, odd, _i32(3, 4), _i32(3), 2)
