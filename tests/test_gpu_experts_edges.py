"""Expert-layer operators on the GPU where they could go wrong.

Tolerances are bounds derived from the arithmetic, given at each test.
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_experts import gen, offsets_of, product64, unpacked  # noqa: E402


@pytest.fixture(scope="module")
def ops():
    from lightgbm_rs_b200 import experts

    yield experts
    experts.check_errors()


# --------------------------------------------------------- rows before the first offset


LEAD = [  # rows before the first offset, counts, tail rows, inner, outer
    (1, [2], 0, 64, 64), (3, [0, 1], 1, 40, 24), (9, [1, 0, 5], 0, 700, 129), (70, [1] * 40, 2, 96, 72),
    (40, [200, 0, 77], 3, 72, 520), (300, [129, 1000], 0, 200, 264), (257, [31, 400], 200, 129, 700),
    (5, [0, 0], 0, 48, 40),
]


@pytest.mark.parametrize("lead,counts,tail,inner,outer", LEAD)
def test_rows_before_the_first_offset_are_zero(ops, lead, counts, tail, inner, outer):
    """A shard of the experts has offsets that do not start at 0. Results go to memory that holds
    NaN: what is not written stays NaN."""
    from lightgbm_rs_b200 import _lib as C

    g, L = gen(lead + inner), C.lib()
    m, E = lead + sum(counts) + tail, len(counts)
    x = torch.randn(m, inner, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(E, outer, inner, generator=g, device="cuda") * inner ** -0.5).to(torch.bfloat16)
    dy = torch.randn(m, outer, generator=g, device="cuda").to(torch.bfloat16)
    off = offsets_of(counts) + lead
    x[:lead], dy[:lead] = math.inf, math.nan  # rows of no expert hold what they like
    st = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    nan = lambda *s: torch.full(s, math.nan, device="cuda", dtype=torch.bfloat16)  # noqa: E731

    y = nan(m, outer)
    n = L.lgbm_b200_experts_matmul_workspace(p(x), inner, None, p(w), m, E, inner, outer)
    ws = torch.empty(max(n, 16), device="cuda", dtype=torch.uint8)
    C.check(L.lgbm_b200_experts_matmul(p(x), m, inner, None, p(w), p(off), 1, m, E, inner, outer,
                                       p(y), p(ws), n, st))
    dx, dw = nan(m, inner), nan(E, outer, inner)
    n = L.lgbm_b200_experts_matmul_backward_workspace(p(dy), outer, p(x), inner, None, p(w), m, E,
                                                      inner, outer, 1, 1)
    ws = torch.empty(max(n, 16), device="cuda", dtype=torch.uint8)
    C.check(L.lgbm_b200_experts_matmul_backward(p(dy), outer, p(x), m, inner, None, p(w), p(off), 1,
                                                1, m, E, inner, outer, p(dx), p(dw), p(ws), n, st))
    q = torch.randint(0, 256, (E, outer, (inner + 31) // 32 * 16), generator=g, device="cuda",
                      dtype=torch.uint8)
    scales = torch.randn(E, outer, -(-inner // 64), generator=g, device="cuda").to(torch.bfloat16)
    y4 = nan(m, outer)
    C.check(L.lgbm_b200_experts_matmul_w4(p(x), m, inner, None, p(q), p(scales), None, 64, p(off), 1,
                                          m, E, inner, outer, p(y4), st))

    inside = slice(lead, m - tail)
    for got, a, b, length in ((y, x, w, inner), (dx, dy, w.transpose(1, 2), outer),
                              (y4, x, unpacked(q, scales, None, inner, 64), inner)):
        assert not got[:lead].any() and not got[m - tail:].any()
        # n products summed in f32 (and scaled by group), and a rounding to bf16
        _, want, mag = product64(a[inside], b, off - lead, None)
        mag = product64(a[inside], b.abs(), off - lead, None)[2]
        lim = 1.1 * length * 2.0 ** -23 * mag + 2.0 ** -8 * want.abs() + 2.0 ** -25
        assert ((got[inside].double() - want).abs() <= lim).all()
    o = off.tolist()
    for e in range(E):
        s = slice(o[e], o[e + 1])
        want, mag = (f(dy[s].double()).T @ f(x[s].double()) for f in (lambda t: t, torch.abs))
        assert ((dw[e].double() - want).abs()
                <= counts[e] * 2.0 ** -23 * mag + 2.0 ** -8 * want.abs()).all()


def test_a_shard_of_the_experts(ops):
    """Experts 2 to 4 of six with their slice of the offsets give their rows of the whole."""
    g = gen(17)
    counts = [50, 3, 70, 0, 20, 9]
    off, m = offsets_of(counts), sum(counts)
    x = torch.randn(m, 72, generator=g, device="cuda").half()
    w = torch.randn(6, 40, 72, generator=g, device="cuda").half()
    whole = ops.grouped_matmul(x, w, off)
    part = ops.grouped_matmul(x, w[2:5], off[2:6])
    lo, hi = int(off[2]), int(off[5])
    assert torch.equal(part[lo:hi], whole[lo:hi])
    assert not part[:lo].any() and not part[hi:].any()
