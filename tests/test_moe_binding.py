"""The compiled entry points of the sparse MLP block's operators, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

from tests.test_decode_binding import _cg, _Elsewhere, _int  # noqa: E402


def _half(*shape, device="cuda:0"):
    return _Elsewhere(device, *shape, dtype=torch.float16)


def test_tensors_on_the_host_are_refused():
    cg, h = _cg(), torch.zeros(2, 64, dtype=torch.float16)
    q = torch.zeros(8, 64, 32, dtype=torch.uint8)
    for call in (lambda: cg.block_norm(h, h, h, 2, 64), lambda: cg.moe_route(h, _int(2, 2), torch.zeros(2, 2), 2, 64, 2),
                 lambda: cg.moe_w4a16_swiglu(h, _int(2, 2), q, h, h, h, 2, 2, 8, 32, 64),
                 lambda: cg.moe_w4a16(h, _int(2, 2), None, q, h, h, h, 2, 1, 8, 64, 64)):
        with pytest.raises(ValueError, match="on the GPU"):
            call()


def test_types_and_sizes_are_checked():
    cg = _cg()
    x, ids = _half(2, 64), _Elsewhere("cuda:0", 2, 2, dtype=torch.int32)
    w = _Elsewhere("cuda:0", 2, 2)
    for bad, why in [((x, x, _Elsewhere("cuda:0", 2, 64), 2, 64), "h_out must be Half"), ((x, x, x, 3, 64), "2 rows"),
                     ((x, x, x, 2, 65), "rows of 64"), ((_half(2, 64, device="cuda:1"), x, x, 2, 64), "residual is on cuda:0")]:
        with pytest.raises(ValueError, match=why):
            cg.block_norm(*bad)
    with pytest.raises(ValueError, match="post_weight must be Half"):
        cg.block_norm(x, x, x, 2, 64, post_weight=_Elsewhere("cuda:0", 64))
    with pytest.raises(ValueError, match="gate must be 64"):
        cg.block_norm(x, x, x, 2, 64, gate=_half(63))
    with pytest.raises(ValueError, match="gate holds 1 rows"):
        cg.block_norm(x, x, x, 2, 64, gate=_half(1, 64))
    with pytest.raises(ValueError, match="weights must be 6"):
        cg.moe_route(x, _Elsewhere("cuda:0", 2, 3, dtype=torch.int32), w, 2, 64, 3)
    with pytest.raises(TypeError, match="ids is not a tensor"):
        cg.moe_route(x, None, w, 2, 64, 2)
    with pytest.raises(ValueError, match="bias must be 64"):
        cg.moe_route(x, ids, w, 2, 64, 2, bias=_Elsewhere("cuda:0", 63))
    q, s = _Elsewhere("cuda:0", 8, 64, 32, dtype=torch.uint8), _half(8, 64, 1)
    up = dict(X=x, ids=ids, W_q=q, W_scale=s, W_zero=s, H=_half(4, 32), T=2, top_k=2, experts=8, I=32, K=64)
    down = dict(H=_half(4, 64), ids=ids, weights=w, W_q=q, W_scale=s, W_zero=s, Y=x, T=2, top_k=2, experts=8, O=64, K=64)
    for f, args in ((cg.moe_w4a16_swiglu, up), (cg.moe_w4a16, down)):
        for name, bad in [("W_q", _Elsewhere("cuda:0", 8, 63, 32, dtype=torch.uint8)), ("W_scale", _half(8, 63)), ("W_zero", _half(8, 63)),
                          ("ids", _Elsewhere("cuda:0", 3, dtype=torch.int32)), ("H", _half(3, 32)), ("ids", _Elsewhere("cuda:0", 2, 2, dtype=torch.int64))]:
            with pytest.raises(ValueError, match=name):
                f(**{**args, name: bad})
        for name in ("ids", "W_q", "W_scale", "W_zero", "H"):
            with pytest.raises(TypeError, match=f"{name} is not a tensor"):
                f(**{**args, name: None})


@pytest.mark.parametrize("T,D", [(2, 64), (3, 1), (5, 7)])
def test_a_flat_gate_is_one_row_or_all_of_them(T, D):
    """A gate of one dimension is a row for all tokens or, as long as all rows, a row for each, as x is;
    of any other length it would be read as something it is not."""
    cg, x = _cg(), _half(T, D)
    for n in (D + 1, T * D - 1, T * D + 1, 2 * T * D):
        if n in (D, T * D):
            continue
        with pytest.raises(ValueError, match=f"gate must be {D} .*not {n}"):
            cg.block_norm(x, x, x, T, D, gate=_half(n), post_weight=_half(D - 1))
    # taken, and refused only for the next argument
    for n in (D, T * D):
        with pytest.raises(ValueError, match="post_weight must be"):
            cg.block_norm(x, x, x, T, D, gate=_half(n), post_weight=_half(D - 1))


def test_entry_points_take_their_number_of_arguments():
    from clove_compute_amd.decode import _b
    for f in (_b.block_norm, _b.moe_route, _b.moe_up, _b.moe_down):
        with pytest.raises(TypeError, match="arguments are wanted"):
            f()
