"""Which kernels the experts' products take, replayed on the host from the kernels' own
moe_plan.hpp: the calls that the GPU tests make reach the kernels that they name."""
import pytest

from tests import _moe_plan as plan


@pytest.mark.parametrize("call", plan.CALLS, ids=plan.named)
def test_calls_reach_the_kernel_they_name(call):
    assert plan.choice(*call[1:])[0] == call[0]


def test_every_kernel_is_reached():
    names = {(c[0], c[1]) for c in plan.CALLS}
    for op in ("up", "down"):
        assert {n for n, o in names if o == op} >= {"many", "some", "thin", "small", "expert2", "expert8", "any"}
        # both ways to list the pairs of a tile
        for shape in ("many", "some", "thin"):
            assert {c[2] * c[3] > 2048 for c in plan.TILES if c[0].split("/")[0] == shape and c[1] == op} == {True, False}
        for shape in ("some", "thin"):
            assert any(c[0].startswith(shape + "/") and c[1] == op for c in plan.TILES)
    assert {n for n, _ in names} >= {"token16x1", "token16x2", "token4x1", "token4x2"}


def test_only_aligned_calls_leave_the_general_kernel():
    for op in ("up", "down"):
        for T, k, E, O, K in [(1, 1, 1, 1, 128), (100, 6, 64, 1408, 2048), (8192, 8, 128, 768, 2048)]:
            assert plan.choice(op, T, k, E, O, K)[0] != "any"
            assert plan.choice(op, T, k, E, O, K, aligned=False)[0] == "any"
            assert plan.choice(op, T, k, E, O, K - 2)[0] == "any"
    # (an expert's weights past the 2^31 bytes that a buffer's offsets reach: of many pairs)
    assert plan.choice("down", 100, 1, 1, 1 << 20, 4096)[0] == "any" != plan.choice("down", 100, 1, 1, (1 << 20) - 1, 4096)[0]


def test_outputs_at_a_time():
    """Whole calls where the products have room in 512 MB and a launch counts the workgroups."""
    for op in ("up", "down"):
        assert plan.choice(op, 8192, 8, 128, 2048, 768)[1] == 2048
    for T, k, O in [(8192, 8, 5000), (32769, 8, 512), (65536, 8, 100000), (1, 1, 512 * 65535 + 700)]:
        chunk = plan.choice("down", T, k, 4, O, 64)[1]
        assert 0 < chunk < O and chunk % 256 == 0 and chunk <= 512 * 65535 and (chunk == 256 or T * k * chunk * 4 <= 512 << 20)
    assert 0 < plan.choice("up", 550, 2, 1024, 262400, 32)[1] < 262400


def test_tokens_at_a_time():
    """As many as 2^19 pairs, and an X below 2^31 bytes, allow, however few columns or many places there are."""
    for op in ("up", "down"):
        for k in (1, 2, 3, 6, 8, 20, 64):
            for K in (0, 2, 8, 10, 30, 32, 64, 4096, 1 << 20, (1 << 24) - 2, 1 << 29, (1 << 30) - 2, 1 << 30, (1 << 31) - 2):
                n, row = plan.tokens_at_a_time(op, k, K), 2 * K * (1 if op == "up" else k)
                assert n * k <= 1 << 19 and n * row < 1 << 31
                assert (n + 1) * k > 1 << 19 or (n + 1) * row >= 1 << 31
