"""GPU: residual_norm and Rotary.rotate on tensors of more than 2^32 bytes and 2^31 elements."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from fleet_moe import _lib, ops, rope  # noqa: E402

BITS = torch.int16


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def noise(*shape):
    """bf16 bits of normal values."""
    return torch.randn(shape, device="cuda").bfloat16().view(BITS)


@pytest.mark.parametrize("rows, width", [(70_000, 32_768), (3_000_000, 1000), (5_000_000, 600),
                                         (20_000_000, 128)])
def test_norms_of_many_rows(rows, width):
    """x and y are the same 1,000 rows over and over, and so are the results; the second and the
    others in more than 2^20 workgroups."""
    torch.manual_seed(1)
    x1, y1 = noise(1000, width), noise(1000, width)
    x = x1.repeat(rows // 1000, 1)
    y = y1.repeat(rows // 1000, 1)
    print(f"[gpu] {rows} rows of {width}", flush=True)
    a1, h1 = ops.residual_norm(x1, y1)
    a, h = ops.residual_norm(x, y, x_out=x)
    for first in range(0, rows, 1000):
        assert torch.equal(a[first: first + 1000], a1) and torch.equal(h[first: first + 1000], h1)


def test_norms_of_rows_far_apart():
    torch.manual_seed(2)
    room = torch.zeros(2**31 + 10_000, dtype=BITS, device="cuda")
    x, y = (torch.as_strided(room, (3, 2048), (2**30, 1), at) for at in (0, 4096))
    x.copy_(noise(3, 2048))
    y.copy_(noise(3, 2048))
    for got, want in zip(ops.residual_norm(x, y, gate=y),
                         ops.residual_norm(x.contiguous(), y.contiguous(), gate=y.contiguous())):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype, tokens, heads, width", [
    (BITS, 200_000, 128, 192), (torch.float32, 100_000, 128, 192), (BITS, 40_000_000, 1, 64)])
def test_rotations_of_many_tokens(dtype, tokens, heads, width):
    """The same 1,000 tokens over and over; the last in more than 2^20 workgroups."""
    torch.manual_seed(3)
    f = rope.frequencies()
    one = noise(1000, heads, width) if dtype == BITS else torch.randn(1000, heads, width, device="cuda")
    pos = torch.arange(1000, dtype=torch.int32, device="cuda") * 7
    r = ops.Rotary(f)
    want = r.rotate(one, pos, at=width - 64)
    x = one.repeat(tokens // 1000, 1, 1)
    print(f"[gpu] {tokens} tokens of {heads} heads", flush=True)
    got = r.rotate(x, pos.repeat(tokens // 1000), at=width - 64)
    for first in range(0, tokens, 1000):
        assert torch.equal(got[first: first + 1000], want)


def test_rotations_of_heads_far_apart():
    torch.manual_seed(4)
    room = torch.zeros(2**31 + 2**30 + 10_000, dtype=BITS, device="cuda")
    r = ops.Rotary(rope.frequencies())
    pos = torch.tensor([3, 500], dtype=torch.int32, device="cuda")
    x = torch.as_strided(room, (2, 2, 64), (2**31, 2**30, 1), 0)
    x.copy_(noise(2, 2, 64))
    out = torch.as_strided(room, (2, 2, 64), (2**30, 2**31, 1), 4096)
    assert torch.equal(r.rotate(x, pos, out=out), r.rotate(x.contiguous(), pos))


def test_more_rows_than_an_int():
    """2^32 + 5 rows of one value (rows of 32 bits: 5) are refused."""
    x = torch.zeros((1, 1), dtype=BITS, device="cuda").expand(2**32 + 5, 1)
    room = torch.zeros(2**32 + 5, dtype=BITS, device="cuda").view(-1, 1)
    with pytest.raises(_lib.FleetMoeError):
        ops.residual_norm(x, h=room)
    assert not room.any()
