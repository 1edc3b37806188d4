"""The key/value cache's operators on the GPU at the ends of their arguments' ranges, against the plain forms."""
import pytest
import torch

from rocknpu_amd import kv
from tests import kv_ref
from tests.test_gpu_kv import DEV, check_attention, ints, random_cache, same_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_new", [5, 1000, 2 ** 31 - 1])
def test_a_bound_above_the_rows(max_new):
    """max_new bounds a sequence's rows: one bound for all of a caller's steps is as good as the step's own."""
    c = random_cache(70, 2, 2, 64, 6)
    r = kv_ref.Ref(c)
    past, cu = [40, 0], [0, 3, 5]
    g = torch.Generator().manual_seed(71)
    k, v = (torch.randn((5, 2, 64), generator=g) for _ in range(2))
    q = torch.randn((5, 6, 64), generator=g)
    r.append(k.numpy(), v.numpy(), past, cu)
    kv.append(c, k.to(DEV), v.to(DEV), ints(past), ints(cu), max_new)
    o = kv.attention(c, q.to(DEV), ints(past), ints(cu), max_new)
    torch.cuda.synchronize()
    same_cache(c, r, [43, 2])
    check_attention(o, r.attention(q.double().numpy(), past, cu), "f32", 64, 43)
    assert torch.equal(o, kv.attention(c, q.to(DEV), ints(past), ints(cu), 3))


@pytest.mark.parametrize("prefix", [2 ** 31 - 1, 2 ** 31 - 31, 2 ** 30, -1, -2 ** 31])
@pytest.mark.parametrize("new", [1, 3, 60])
@pytest.mark.parametrize("lost", [0, 4])
def test_prefixes_beyond_every_position(prefix, new, lost):
    """With a window too: a prefix of 2^31 - 1 keeps all keys, a negative one none."""
    past, cu = [700, 90], [0, new, 2 * new]
    c = random_cache(72, 2, 2, 64, 26, [lost, 0], past)
    q = torch.randn((2 * new, 8, 64), generator=torch.Generator().manual_seed(73))
    wo = torch.full_like(c.weights, float("nan")) if new < 60 else None
    o = kv.attention(c, q.to(DEV), ints(past), ints(cu), new, window=40, prefix=ints([prefix] * 2), weights_out=wo)
    r = kv_ref.Ref(c)
    want = r.attention(q.double().numpy(), past, cu, window=40, prefix=[prefix] * 2)
    check_attention(o, want, "f32", 64, 760)
    if wo is not None:
        assert (abs(wo.cpu().double().numpy() - r.weights - want[3]) <= 1e-4).all()
