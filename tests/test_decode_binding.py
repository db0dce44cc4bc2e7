"""The compiled entry points of the decode step's operators, without a GPU: they load
beside the library and refuse what they can judge on the host."""
import pytest

torch = pytest.importorskip("torch")


def _cg():
    import clove_compute_amd as cg
    return cg


def _int(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_tensors_on_the_host_are_refused():
    cg = _cg()
    x = torch.ones(2, 64)
    with pytest.raises(ValueError, match="on the GPU"):
        cg.penalize_logits(x, x, 2, 64)
    h = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="on the GPU"):
        cg.qk_norm_rope(h, None, None, x, x, _int(2), h, 2, 1, 1, 16)
    with pytest.raises(ValueError):
        cg.KVCache(torch.zeros(1, 1, 4, 8, dtype=torch.float16), torch.zeros(1, 1, 4, 8, dtype=torch.float16))


def test_what_is_no_tensor_or_number_is_refused():
    cg = _cg()
    x = torch.ones(2, 64)
    for bad in (None, 3, [1.0], "x"):
        with pytest.raises(TypeError, match="logits is not a tensor"):
            cg.penalize_logits(bad, x, 2, 64)
    with pytest.raises(TypeError):
        cg.penalize_logits(x, x, 2.5, 64)
    with pytest.raises(OverflowError):
        cg.penalize_logits(x, x, 2 ** 31, 64)
    with pytest.raises(AttributeError):
        cg.paged_attention(x, object(), _int(2, 1), _int(2), x, 2, 1, 4)


def test_entry_points_take_their_number_of_arguments():
    from clove_compute_amd import decode
    for f in (decode._b.rope, decode._b.attend, decode._b.evict, decode._b.penalize):
        with pytest.raises(TypeError, match="arguments are wanted"):
            f()


def test_caches_of_pages_that_lie_on_each_other_are_refused():
    """An expanded tensor's pages are all one: the library would take its distance, 0,
    for that of dense pages and go past its end."""
    cg = _cg()
    page = torch.zeros(1, 2, 4, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="lie apart"):
        cg.KVCache(page.expand(5, -1, -1, -1), page.expand(5, -1, -1, -1))
    near = torch.zeros(200, dtype=torch.float16).as_strided((3, 2, 4, 8), (63, 32, 8, 1))
    with pytest.raises(ValueError, match="lie apart"):
        cg.KVCache(near, near)
    for fine in (page.expand(1, -1, -1, -1), torch.zeros(3, 2, 4, 8, dtype=torch.float16), torch.zeros(3, 2, 2, 4, 8, dtype=torch.float16)[:, 1]):
        with pytest.raises(ValueError, match="on the GPU"):  # (nothing else is wrong with it)
            cg.KVCache(fine, fine)


class _Elsewhere(torch.Tensor):
    """A tensor of a device that need not be there (it has no memory: the checks come first)."""

    @staticmethod
    def __new__(cls, device, *shape, dtype=torch.float32):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device=device)

    @classmethod
    def __torch_dispatch__(cls, *args, **kwargs):
        raise AssertionError("only looked at")


def test_tensors_of_two_devices_are_refused():
    cg = _cg()
    x, y = _Elsewhere("cuda:0", 2, 64), _Elsewhere("cuda:1", 2, 64)
    with pytest.raises(ValueError, match="out is on cuda:1, other tensors are on cuda:0"):
        cg.penalize_logits(x, y, 2, 64)
    h, n = _Elsewhere("cuda:1", 2, 5, dtype=torch.int32), _Elsewhere("cuda:0", 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="history is on cuda:1"):
        cg.penalize_logits(x, x, 2, 64, history=h, history_lens=n)
    q = _Elsewhere("cuda:0", 2, 64, dtype=torch.float16)

    class Cache:  # what a KVCache of the other device hands on
        from clove_compute_amd.decode import _CacheAt
        head_dim, _c = 64, _CacheAt(0x1000, 0x2000, 0, 8, 16, 1, 64, 0, 1)
        import ctypes
        _at = ctypes.addressof(_c)

    with pytest.raises(ValueError, match="q is on cuda:0, other tensors are on cuda:1"):
        cg.paged_attention(q, Cache, n, n, q, 2, 1, 16)


def test_a_cache_of_two_devices_is_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        k, v = (torch.empty(4, 2, 16, 64, dtype=torch.float16, device=d) for d in ("cuda:0", "cuda:1"))
    with pytest.raises(ValueError, match="the same one"):
        _cg().KVCache(k, v)
