"""How near the kernels come to the chain in 64 bits, next to the oracle's
chain in f32 (the same steps, products and sums in f32).

The wide route holds an operand in two f16 planes: 2^-23 of it is lost at most
where f32 loses 2^-24, in each of the two, and the product of the two lows,
2^-22, is left out: six of f32's roundings of a product's value, of which f32
itself has two of the operands (made by the product before) and those of its
sums.  Its sums run over 32 places at a time in f32, as the oracle's do.  The
error is held to eight times the oracle's.
"""
import pytest
import torch

from flink_parameter_server_amd import ops


def exact(u, steps=5, coeffs=ops.MUON_COEFFS, eps=1e-7):
    a, b, c = coeffs
    x = u.double()
    x = x / (x.flatten(1).norm(dim=1)[:, None, None] + eps)
    if x.shape[1] > x.shape[2]:
        return exact(u.mT, steps, coeffs, eps).mT
    for _ in range(steps):
        g = x @ x.mT.contiguous()
        x = a * x + (b * g + c * g @ g) @ x
    return x


def matrices(kind, b, m, n):
    g = torch.Generator().manual_seed(m * n)
    x = torch.randn(b, m, n, generator=g)
    if kind == "decay":  # a few strong directions
        r = min(m, n, 8)
        left = torch.randn(b, m, r, generator=g) / torch.arange(1, r + 1)
        x = torch.bmm(left, torch.randn(b, r, n, generator=g)) + 0.05 * x
    elif kind == "steep":  # four directions a thousand times the others
        x = 1e-3 * x + torch.bmm(torch.randn(b, m, 4, generator=g),
                                 torch.randn(b, 4, n, generator=g))
    return x


SIZES = [(1, 3, 5), (2, 33, 70), (1, 2500, 48), (1, 48, 2500), (1, 65, 65),
         (2, 130, 100), (1, 600, 128), (1, 128, 900), (1, 1200, 200),
         (2, 200, 300), (1, 400, 520), (3, 300, 1001), (1, 700, 513),
         (1, 1024, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "decay", "steep"])
@pytest.mark.parametrize("b,m,n", SIZES)
def test_f32(kind, b, m, n):
    x = matrices(kind, b, m, n)
    want = exact(x)
    f32 = ops.orthogonalize(x)
    got = ops.orthogonalize(x.cuda()).cpu()
    for k in range(b):
        near = float((f32[k].double() - want[k]).norm())
        assert float((got[k].double() - want[k]).norm()) <= 8 * near


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "decay", "steep"])
@pytest.mark.parametrize("b,m,n", SIZES)
def test_f16(kind, b, m, n):
    """Rounded once: as far off as the exact result's own rounding, and what
    f32 results may be."""
    x = matrices(kind, b, m, n).half()
    want = exact(x)
    f32 = ops.orthogonalize(x.float())
    got = ops.orthogonalize(x.cuda()).cpu()
    for k in range(b):
        near = float((f32[k].double() - want[k]).norm())
        rounding = float((want[k].half().double() - want[k]).norm())
        # a value that goes to the other neighbour is off by no more than
        # the rounding of a value next to the middle, and what moved it
        assert float((got[k].double() - want[k]).norm()) <= \
            rounding + 8 * near


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(300, 20), (700, 100), (100, 700),
                                 (300, 140)])
def test_table(m, n):
    """A table's step, its weights zero before it: as f32 results may be, and
    the roundings of U, the rate and the product."""
    x = matrices("decay", 1, m, n)
    f32 = ops.orthogonalize(x)[0]
    want = exact(x)[0]
    near = float((f32.double() - want).norm())
    table = torch.zeros(m, n, device="cuda")
    ops.apply_muon(table, torch.zeros_like(table),
                   torch.arange(m, device="cuda"), x[0].cuda(), 0.5, mu=0.0,
                   sorted_unique=True)
    rate = 0.5 * max(1.0, m / n) ** 0.5
    off = float((table.cpu().double() / -rate - want).norm())
    assert off <= 8 * near + 3 * 2.0 ** -24 * float(want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,m,n", [(3, 40, 60), (2, 3000, 40), (3, 600, 128),
                                   (3, 200, 150), (4, 512, 800)])
def test_neighbours_do_not_matter(b, m, n, dtype):
    """A matrix's result in a batch of a given length is the same to the bit
    whatever the others hold."""
    x = matrices("decay", b, m, n).to(dtype).cuda()
    want = ops.orthogonalize(x)[1].clone()
    for value in (None, 0.0, float("nan"), float("inf"), 1e-30):
        y = x.clone()
        others = [k for k in range(b) if k != 1]
        y[others] = torch.randn_like(y[others]) if value is None else value
        assert torch.equal(ops.orthogonalize(y)[1], want), value


@pytest.mark.gpu
@pytest.mark.parametrize("b,m,n", [(9, 64, 66), (6, 128, 520), (5, 300, 1001)])
def test_alone_and_in_a_batch(b, m, n):
    """How many matrices there are may choose the route and the order of the
    sums: the results are each as near as f32's."""
    x = matrices("decay", b, m, n)
    want = exact(x)
    f32 = ops.orthogonalize(x)
    for k in (0, b - 1):
        near = float((f32[k].double() - want[k]).norm())
        got = ops.orthogonalize(x[k:k + 1].cuda())[0].cpu()
        assert float((got.double() - want[k]).norm()) <= 8 * near


def low_rank(kind, m, n):
    g = torch.Generator().manual_seed(m + n)
    if kind == "ones":  # every value is rounded alike
        return torch.ones(1, m, n) / 3
    if kind == "column":
        x = torch.zeros(1, m, n)
        x[:, :, n // 2] = torch.randn(m, generator=g)
        return x
    if kind == "row":
        x = torch.zeros(1, m, n)
        x[:, m // 2] = torch.randn(n, generator=g)
        return x
    return torch.bmm(torch.randn(1, m, 2, generator=g),
                     torch.randn(1, 2, n, generator=g))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["ones", "column", "row", "rank2"])
@pytest.mark.parametrize("m,n", [(40, 60), (6040, 32), (32, 6040), (900, 128),
                                 (300, 900), (900, 300), (400, 520),
                                 (520, 400), (1000, 700)])
def test_low_rank(kind, m, n):
    """Singular values of zero: the chain multiplies what lies there by
    a^5 = 485.  P is 485 (1 - v v') + p v v', whose values' sizes are a matrix
    of norm 970 at most, and |X| is 1.  P U is made of values of P and U that
    are 2^-24 off, without the product of their lows (2^-24), with three f32
    additions for 32 of s places and a few at the ends: all of them 970 times
    2^-24.  Steps on X make as many of them, each multiplied by what follows:
    no more than five times that."""
    x = low_rank(kind, m, n)
    s = min(m, n)
    limit = 970 * (6 + 3 * (s // 32 + 1)) * 2.0 ** -24
    if not (s <= 64 or s <= 320 and max(m, n) >= 3 * s):
        limit *= 5
    off = float((ops.orthogonalize(x.cuda()).cpu().double()
                 - exact(x)).norm())
    assert off <= limit
