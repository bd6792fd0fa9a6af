"""Routing operators (include/mpkexperts.h) on a B200 against their FP64 definitions (tests/experts_ref.py).

Choices and plans are compared exactly.  Tolerances of computed numbers: the rounding to the output's type (half
a step, eps / 2 relative) plus the FP32 arithmetic behind it, stated beside each check.
"""

import numpy as np
import pytest

import experts_ref as R

torch = pytest.importorskip("torch")
import mpkmeans_b200 as M  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half of the type's least subnormal step: the absolute error of rounding a tiny value."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def f64(t):
    return t.double().cpu().numpy()


def normal(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# ------------------------------------------------------------------ route --

def weights_close(got, want, x, ids):
    """exp of an argument rounded in FP32 (relative error |x - max| u), a few roundings, a sum of up to 1024 terms by
    32 per lane and 5 levels."""
    finite = np.where(np.isfinite(x), x, 0)
    spread = 2 * np.abs(finite).max(1, keepdims=True) + 64 if x.shape[0] else np.zeros((0, 1))
    assert np.all(np.abs(got - want) <= spread * U32 * np.abs(want) + 1e-37)


def check_route(x, top_k, bias=None, **kw):
    ids, w = M.route(x, top_k, bias=bias, **kw)
    want_ids, want_w = R.route(f64(x), top_k, bias=None if bias is None else f64(bias), **kw)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    weights_close(f64(w), want_w, f64(x), want_ids)
    return ids, w


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n,experts,top_k", [(1, 1, 1), (1, 64, 6), (3, 2, 2), (37, 33, 5), (130, 256, 8), (9, 1000, 32),
                                             (5, 1024, 1), (64, 8, 8), (2, 40, 32)])
def test_route(n, experts, top_k, score, dtype):
    x = normal(n + experts, n, experts, dtype=TYPES[dtype], scale=2.0)
    bias = normal(7, experts, scale=0.1)
    for renormalize in (True, False):
        check_route(x, top_k, score=score, renormalize=renormalize, scale=1.25)
        check_route(x, top_k, bias=bias, score=score, renormalize=renormalize)


@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(256, 8, 4, 8), (64, 4, 1, 6), (96, 32, 3, 4), (60, 5, 2, 7),
                                                             (16, 16, 4, 4), (1024, 2, 1, 3), (18, 3, 3, 18), (33, 11, 2, 6)])
def test_route_groups(experts, groups, top_groups, top_k, score, group_score):
    kw = dict(groups=groups, top_groups=top_groups, group_score=group_score, score=score)
    x = normal(experts, 53, experts, scale=1.5)
    check_route(x, top_k, **kw)
    check_route(x, top_k, bias=normal(5, experts, scale=0.2), renormalize=False, **kw)
    check_route(x.bfloat16(), top_k, bias=torch.zeros(experts, device="cuda"), **kw)        # ties of the coarse type


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_near_ties_are_decided_exactly(score):
    """Choice values closer than FP32 tells apart: logits one step from each other, with a bias."""
    base = torch.linspace(-1, 1, 64)
    x = torch.stack([torch.nextafter(base, base + 1) if i % 2 else base for i in range(2)])
    x = torch.cat([x, x.roll(1, 0)], 1).repeat(8, 1).cuda().contiguous()
    bias = torch.zeros(128, device="cuda")
    check_route(x, 16, score=score, bias=bias)
    check_route(x, 32, score=score, bias=bias)                                             # no lane holds the first loser
    check_route(x, 16, score=score, bias=bias, groups=8, top_groups=3, group_score="top2")
    check_route(x, 16, score=score, groups=8, top_groups=3, group_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_near_groups_are_decided_exactly(score):
    """Groups whose sums differ by less than FP32 scores are off, with biases that cancel inside a group."""
    gen = np.random.default_rng(2)
    base = gen.normal(size=(400, 8))
    x = np.concatenate([base + gen.integers(-3, 4, size=base.shape) * 2.0 ** -23 * np.abs(base) for _ in range(4)], 1)
    x = torch.from_numpy(x.astype(np.float32)).cuda()
    for size in (0.0, 1.0, 20.0):
        bias = torch.from_numpy(np.tile(size * gen.normal(size=8), 4).astype(np.float32)).cuda()
        for group_score in ("max", "top2"):
            check_route(x, 6, score=score, bias=bias, groups=4, top_groups=2, group_score=group_score)


def test_route_saturated_scores_follow_the_logits():
    """Sigmoids that FP64 rounds to one another: the order stays the logits', in rows decided in FP64 too."""
    x = torch.full((4, 64), -1.0, device="cuda")
    x[:, 3], x[:, 9], x[:, 40], x[:, 41] = 50.0, 60.0, 70.0, 45.0
    x[1, 16:18], x[1, 32:34] = 30.0, 30.0                          # groups that tie
    for k in (3, 4):
        ids, _ = M.route(x, k, score="sigmoid", groups=4, top_groups=2, group_score="top2")
        rows = [x[t, ids[t].long()].tolist() for t in range(4)]
        assert all(r == sorted(r, reverse=True) for r in rows)


def test_route_ties_go_to_the_lowest_index():
    x = torch.zeros(4, 100, device="cuda")
    x[1, 50:] = 1.0
    x[2] = -0.0
    x[2, 3] = 0.0
    x[3] = torch.finfo(torch.float32).min                      # the lowest value is no mask
    ids, w = check_route(x, 5)
    assert ids.tolist() == [[0, 1, 2, 3, 4], [50, 51, 52, 53, 54], [0, 1, 2, 3, 4], [0, 1, 2, 3, 4]]
    assert torch.all((w - 0.2).abs() <= 4 * U32)
    check_route(x, 5, bias=torch.zeros(100, device="cuda"))
    check_route(x, 5, score="sigmoid", groups=4, top_groups=2, group_score="top2")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_masks(score, dtype):
    x = normal(1, 40, 48, dtype=TYPES[dtype])
    x[:, 5] = float("-inf")
    x[3] = float("-inf")                                        # nothing left
    x[4, 1:] = float("-inf")                                    # one expert left for four slots
    x[5, 8:] = float("-inf")
    x[6, :24] = torch.finfo(TYPES[dtype]).min
    for kw in (dict(), dict(renormalize=False), dict(groups=6, top_groups=2, group_score="top2"),
               dict(groups=6, top_groups=2, group_score="max"), dict(bias=normal(2, 48, scale=0.1))):
        ids, w = check_route(x, 4, score=score, **kw)
        assert torch.all(ids[3] == -1) and torch.all(w[3] == 0)
        assert ids[4].tolist() == [0, -1, -1, -1]
    bias = torch.zeros(48, device="cuda")
    bias[:47] = float("-inf")                                   # a bias masks as well
    ids, _ = check_route(x[:3], 2, score=score, bias=bias)
    assert ids.tolist() == [[47, -1]] * 3


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_nan_rows_stay_inside(score):
    x = normal(1, 6, 48)
    x[1, 7] = float("nan")
    x[2].view(torch.int32).fill_(0xffc00000 - 2 ** 32)             # NaN with the sign bit set
    assert torch.signbit(x[2]).all()
    for kw in (dict(), dict(renormalize=False), dict(bias=normal(2, 48, scale=0.1)),
               dict(groups=6, top_groups=2, group_score="top2")):
        ids, w = M.route(x, 4, score=score, **kw)
        assert int(ids.min()) >= -1 and int(ids.max()) < 48
        assert torch.isnan(w[1]).any() and torch.isnan(w[2]).all()
        rest = [0, 3, 4, 5]
        want, ww = R.route(f64(x)[rest], 4, score=score, **{k: f64(v) if k == "bias" else v for k, v in kw.items()})
        assert np.array_equal(ids.cpu().numpy()[rest], want)
    x = normal(1, 2, 48)
    x[1, 3] = float("inf")
    ids, w = M.route(x, 4, score=score)
    assert ids[1, 0] == 3 and (torch.isnan(w[1]).all() if score == "softmax" else torch.isfinite(w[1]).all())


def test_route_tiny_scores_keep_their_ratios():
    x = torch.full((2, 8), -200.0, device="cuda")
    x[0, 2], x[0, 5] = -150.0, -150.5
    x[1, 1], x[1, 4] = -61.0, -62.0
    check_route(x, 2, score="sigmoid")
    check_route(x, 2, score="softmax")
    g = normal(1, 2, 2)
    ids, _ = M.route(x, 2, score="sigmoid")
    want = R.route_grad(f64(g), f64(x), ids.cpu().numpy(), score="sigmoid")
    got = f64(M.route_grad(g, x, ids, score="sigmoid"))
    assert np.all(np.abs(got - want) <= 400 * U32 * np.abs(f64(g)).max())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_route_strided_rows(dtype):
    assert M.route(normal(3, 0, 8, dtype=TYPES[dtype]), 2)[0].shape == (0, 2)
    big = normal(3, 20, 80, dtype=TYPES[dtype])
    check_route(big[:, 3:63], 5)
    check_route(big[::2, :60], 5, score="sigmoid", bias=normal(5, 60, scale=0.1))


def grad_tolerance(want, g, x, dtype, scale):
    """dl is a product of a weight (relative error as in weights_close) and a difference of gradients whose rounding is
    relative to the row's largest gradient."""
    spread = 2 * np.abs(np.where(np.isfinite(x), x, 0)).max(1, keepdims=True) + 128
    return half_step(dtype) * np.abs(want) + 4 * spread * U32 * scale * np.abs(g).max(1, keepdims=True) + least(dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("n,experts,top_k", [(1, 1, 1), (1, 64, 6), (70, 60, 4), (33, 256, 8), (6, 1024, 32), (5, 31, 31)])
def test_route_grad(n, experts, top_k, renormalize, score, dtype):
    x = normal(experts, n, experts, dtype=TYPES[dtype], scale=1.5)
    if experts > 40:
        x[:, ::3] = float("-inf")
        x[0] = float("-inf") if n > 1 else x[0]
    kw = dict(score=score, renormalize=renormalize, scale=1.5)
    ids, _ = M.route(x, top_k, **kw)
    g = normal(9, n, top_k)
    got = f64(M.route_grad(g, x, ids, **kw))
    want = R.route_grad(f64(g), f64(x), ids.cpu().numpy(), **kw)
    assert np.all(np.abs(got - want) <= grad_tolerance(want, f64(g), f64(x), TYPES[dtype], 1.5))


def test_route_grad_of_any_ids():
    """The same expert twice, ids out of range, a strided output whose padding stays."""
    x = normal(1, 4, 20)
    ids = torch.tensor([[3, 3, 5], [-1, -1, -1], [0, 19, -1], [7, 20, -5]], dtype=torch.int32, device="cuda")
    g = normal(2, 4, 3)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            out = torch.full((4, 32), 7.0, device="cuda")
            M.route_grad(g, x, ids, score=score, renormalize=renormalize, out=out[:, :20])
            want = R.route_grad(f64(g), f64(x), ids.cpu().numpy(), score=score, renormalize=renormalize)
            assert np.all(np.abs(f64(out)[:, :20] - want) <= grad_tolerance(want, f64(g), f64(x), torch.float32, 1.0))
            assert torch.all(out[:, 20:] == 7.0)


def test_route_grad_against_differences():
    x = normal(11, 3, 10, scale=0.7)
    g = normal(12, 3, 3)
    for score in ("softmax", "sigmoid"):
        ids, _ = M.route(x, 3, score=score)
        got = f64(M.route_grad(g, x, ids, score=score))
        h = 2.0 ** -7
        for j in range(10):
            up, down = x.clone(), x.clone()
            up[:, j] += h
            down[:, j] -= h
            iu, wu = M.route(up, 3, score=score)
            idn, wd = M.route(down, 3, score=score)
            if not (torch.equal(iu, ids) and torch.equal(idn, ids)):
                continue
            d = ((f64(wu) - f64(wd)) * f64(g)).sum(1) / (2 * h)
            # central differences: third derivatives of order one times h^2 / 6, and FP32 weights over 2 h
            assert np.all(np.abs(d - got[:, j]) <= (h * h + 100 * U32 / h) * np.abs(f64(g)).sum(1))


# ------------------------------------------------------------------- plan --

def random_ids(seed, n, top_k, experts, dropped=0.0, skew=0.0):
    rng = np.random.default_rng(seed)
    p = np.exp(skew * rng.normal(size=experts))
    ids = rng.choice(experts, size=(n, top_k), p=p / p.sum()).astype(np.int32)
    ids[rng.random((n, top_k)) < dropped] = -1
    return torch.from_numpy(ids).cuda()


@pytest.mark.parametrize("n,top_k,experts,dropped", [(0, 2, 5, 0), (1, 1, 1, 0), (1, 8, 64, 0), (1, 1, 1024, 0), (7, 3, 33, 0.3),
                                                     (500, 4, 16, 1.0), (2731, 6, 160, 0.1), (16384, 1, 8, 0), (16385, 1, 3, 0.1),
                                                     (9000, 8, 256, 0.05), (4097, 17, 1000, 0.2), (131072, 2, 64, 0), (8000, 1, 1024, 0.1), (8192, 1, 1, 0)])
def test_plan(n, top_k, experts, dropped):
    ids = random_ids(n + experts, n, top_k, experts, dropped, 1.0)
    p = M.expert_plan(ids, experts)
    want = R.plan(ids.cpu().numpy(), experts)
    for got, w in zip((p.offsets, p.order, p.pos), want):
        assert np.array_equal(got.cpu().numpy(), w)


def test_plan_drops_ids_out_of_range():
    ids = torch.tensor([[0, 4], [-7, 2 ** 31 - 1], [3, 3], [-2 ** 31, 1]], dtype=torch.int32, device="cuda")
    p = M.expert_plan(ids, 4)
    assert p.offsets.tolist() == [0, 1, 2, 2, 4]
    assert p.order.tolist() == [0, 7, 4, 5, -1, -1, -1, -1]
    assert p.pos.tolist() == [[0, -1], [-1, -1], [2, 3], [-1, 1]]


# --------------------------------------------------------------- products --

def product_tolerance(want, magnitude, length, dtype):
    """One rounding to the type, and FP32 sums of `length` exact products, each addition off by at most one step of the
    running sum (the tensor cores truncate): 2^-23 of the sum of magnitudes each."""
    return half_step(dtype) * (np.abs(want) + length * 2 * U32 * magnitude) + length * 2 * U32 * magnitude + least(dtype)


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    """Every test ends with the products' device status clear."""
    yield
    assert M.lib().mpkDebugExpertStatus(1) == 0


def setup_products(seed, n, top_k, experts, k, width, dtype, gather, dropped, skew):
    ids = random_ids(seed, n, top_k, experts, dropped, skew)
    plan = M.expert_plan(ids, experts)
    off, order, _ = R.plan(ids.cpu().numpy(), experts)
    x = normal(seed + 1, n if gather else n * top_k, k, dtype=dtype)
    w = normal(seed + 2, experts, width, k, dtype=dtype, scale=k ** -0.5)
    g = normal(seed + 3, n * top_k, width, dtype=dtype)
    xs = R.gathered(f64(x), order, top_k) if gather else f64(x)
    return plan, off, x, xs, w, g


def check_products(plan, off, x, xs, w, g, gather, dtype, outs=(None, None, None)):
    k, width = w.shape[2], w.shape[1]
    kept = off[-1]
    y = M.expert_gemm(x, w, plan, gather=gather, out=outs[0])
    want, mag = R.gemm(xs, f64(w), off), R.gemm(np.abs(xs), np.abs(f64(w)), off)
    assert np.all(np.abs(f64(y) - want) <= product_tolerance(want, mag, k, dtype))
    assert torch.all(y[kept:] == 0)
    dx = M.expert_gemm_grad_x(g, w, plan, out=outs[1])
    wt = f64(w).transpose(0, 2, 1)
    want, mag = R.gemm(f64(g), wt, off), R.gemm(np.abs(f64(g)), np.abs(wt), off)
    assert np.all(np.abs(f64(dx) - want) <= product_tolerance(want, mag, width, dtype))
    assert torch.all(dx[kept:] == 0)
    dw = M.expert_gemm_grad_w(g, x, plan, gather=gather, out=outs[2])
    want, mag = R.gemm_grad_w(f64(g), xs, off), R.gemm_grad_w(np.abs(f64(g)), np.abs(xs), off)
    most = int((off[1:] - off[:-1]).max())
    assert np.all(np.abs(f64(dw) - want) <= product_tolerance(want, mag, most, dtype))
    for e in np.flatnonzero(off[1:] == off[:-1]):
        assert torch.all(dw[e] == 0)


SHAPES = [  # n, top_k, experts, k, width, dropped, skew
    (1, 1, 1, 8, 8, 0, 0),
    (1, 8, 64, 256, 136, 0, 0),
    (1, 2, 4, 64, 128, 0.5, 0),
    (5, 2, 16, 1024, 72, 0, 1),
    (17, 3, 7, 200, 264, 0.1, 1),
    (96, 6, 64, 128, 256, 0, 1),
    (130, 2, 3, 72, 520, 0, 0.5),
    (300, 4, 5, 136, 128, 0.2, 2),
    (513, 2, 2, 64, 640, 0, 0),
    (700, 1, 1, 384, 384, 0, 0),
    (64, 4, 8, 8, 1000, 1.0, 0),
    (999, 2, 40, 320, 48, 0.05, 1),
    (2000, 2, 1000, 64, 64, 0.05, 1),
    (2100, 4, 2, 64, 96, 0, 0.5),
    (16, 1, 1, 264, 136, 0, 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("n,top_k,experts,k,width,dropped,skew", SHAPES)
def test_products(n, top_k, experts, k, width, dropped, skew, gather, dtype):
    s = setup_products(n + k, n, top_k, experts, k, width, TYPES[dtype], gather, dropped, skew)
    check_products(*s, gather, TYPES[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("n,top_k,experts,k,width", [(1, 1, 1, 1, 1), (1, 4, 8, 37, 19), (33, 2, 5, 101, 67), (200, 3, 4, 130, 66),
                                                     (130, 2, 3, 64, 33), (70, 2, 3, 33, 64)])
def test_products_odd_widths(n, top_k, experts, k, width, gather, dtype):
    """Rows that do not start on 16-byte boundaries."""
    s = setup_products(n + k, n, top_k, experts, k, width, TYPES[dtype], gather, 0.1, 1)
    check_products(*s, gather, TYPES[dtype])


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("pad", [8, 3])
@pytest.mark.parametrize("n,top_k,experts,k,width", [(150, 2, 5, 136, 264), (16, 1, 1, 64, 72), (7, 2, 4, 88, 40), (60, 2, 12, 64, 64)])
def test_products_strides(n, top_k, experts, k, width, gather, pad):
    """Operands and outputs inside larger buffers; nothing beside the results is written."""
    dtype = torch.bfloat16
    plan, off, x, xs, w, g = setup_products(4, n, top_k, experts, k, width, dtype, gather, 0.1, 1)

    def inside(t):
        big = torch.full([d + (2 if i < t.dim() - 1 else pad) for i, d in enumerate(t.shape)], float("nan"), dtype=dtype,
                         device="cuda")
        view = big[tuple(slice(0, d) for d in t.shape)]
        view.copy_(t)
        return view

    outs = []
    for shape in ((n * top_k, width), (n * top_k, k), (experts, width, k)):
        outs.append(torch.full([d + (2 if i < len(shape) - 1 else pad) for i, d in enumerate(shape)], 7.0, dtype=dtype,
                               device="cuda"))
    views = [o[tuple(slice(0, d) for d in shape)] for o, shape in
             zip(outs, ((n * top_k, width), (n * top_k, k), (experts, width, k)))]
    check_products(plan, off, inside(x), xs, inside(w), inside(g), gather, dtype, views)
    for o, v in zip(outs, views):
        v.fill_(7.0)
        assert torch.all(o == 7.0)


@pytest.mark.parametrize("n", [4, 200])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_products_keep_experts_apart(value, n):
    """Non-finite rows of one expert reach neither another expert's rows nor its gradient; non-finite rows behind the
    last routed one reach nothing."""
    dtype, top_k, experts, k, width = torch.bfloat16, 2, 3, 192, 136
    ids = random_ids(1, n, top_k, experts, 0.0, 0.0)
    ids[0, 0] = -1
    plan = M.expert_plan(ids, experts)
    off, order, _ = R.plan(ids.cpu().numpy(), experts)
    x, g = normal(2, n * top_k, k, dtype=dtype), normal(4, n * top_k, width, dtype=dtype)
    w = normal(3, experts, width, k, dtype=dtype, scale=k ** -0.5)
    a, b = int(off[1]), int(off[2])
    clean = np.r_[0:a, b:off[-1]]
    zeroed = [t.clone() for t in (x, g)]
    for t, z in zip((x, g), zeroed):
        t[a:b] = value
        t[off[-1]:] = value
        z[a:b] = 0
        z[off[-1]:] = 0
    x64, g64, w64 = (f64(t) for t in (*zeroed, w))
    wt = w64.transpose(0, 2, 1)
    for out, rows, m, length in ((M.expert_gemm(x, w, plan, gather=False), x64, w64, k),
                                 (M.expert_gemm_grad_x(g, w, plan), g64, wt, width)):
        want, mag = R.gemm(rows, m, off), R.gemm(np.abs(rows), np.abs(m), off)
        assert np.all(np.abs(f64(out) - want)[clean] <= product_tolerance(want, mag, length, dtype)[clean])
        assert torch.all(out[off[-1]:] == 0)
    dw = f64(M.expert_gemm_grad_w(g, x, plan, gather=False))
    want, mag = R.gemm_grad_w(g64, x64, off), R.gemm_grad_w(np.abs(g64), np.abs(x64), off)
    assert np.all(np.abs(dw - want)[[0, 2]] <= product_tolerance(want, mag, int(off[-1]), dtype)[[0, 2]])


@pytest.mark.parametrize("width,k", [(64, 72), (33, 35)])
def test_products_bad_plans_stay_inside(width, k):
    """Offsets and entries that no plan holds give meaningless rows, but none outside the buffers."""
    n, top_k, experts = 40, 2, 4
    rows = n * top_k
    bad = [([0, 100000, -5, 7, 2 ** 31 - 1], 2 ** 31 - 1), ([50, 40, 30, 20, 10], -2 ** 31), ([-1, -1, 90, 90, 80], 12345)]
    for offsets, entry in bad:
        off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        order = torch.full((rows,), entry, dtype=torch.int32, device="cuda")
        pos = torch.full((n, top_k), entry, dtype=torch.int32, device="cuda")
        plan = M.ExpertPlan(off, order, pos)
        x, w = normal(1, n, k, dtype=torch.float16), normal(2, experts, width, k, dtype=torch.float16)
        g = normal(3, rows, width, dtype=torch.float16)
        guard = torch.full((3, rows + 8, 128), 7.0, dtype=torch.float16, device="cuda")
        M.expert_gemm(x, w, plan, out=guard[0, 4:-4, :width])
        M.expert_gemm_grad_x(g, w, plan, out=guard[1, 4:-4, :k])
        M.expert_gemm_grad_w(g, x, plan)
        M.expert_combine(g, plan)
        M.expert_combine_grad(normal(4, n, width, dtype=torch.float16), g, plan, out=guard[2, 4:-4, :width])
        torch.cuda.synchronize()
        for i, c in enumerate((width, k, width)):
            assert torch.all(guard[i, :4] == 7) and torch.all(guard[i, -4:] == 7) and torch.all(guard[i, :, c:] == 7)


def test_products_without_rows():
    plan = M.expert_plan(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 4)
    assert plan.offsets.tolist() == [0] * 5
    x, w = normal(1, 0, 64, dtype=torch.float16), normal(2, 4, 32, 64, dtype=torch.float16)
    assert M.expert_gemm(x, w, plan).shape == (0, 32)
    assert M.expert_gemm_grad_x(normal(1, 0, 32, dtype=torch.float16), w, plan).shape == (0, 64)
    dw = M.expert_gemm_grad_w(normal(1, 0, 32, dtype=torch.float16), x, plan, out=torch.ones_like(w))
    assert torch.all(dw == 0)
    assert M.expert_combine(normal(1, 0, 32), plan).shape == (0, 32)


# ---------------------------------------------------------------- combine --

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,top_k,width,dropped", [(1, 1, 1, 0), (1, 8, 2048, 0), (3, 2, 17, 0.5), (50, 9, 264, 0.1), (33, 4, 4104, 0),
                                                   (200, 3, 8, 1.0), (7, 20, 100, 0.2), (2500, 2, 12, 0.1)])
def test_combine_and_grad(n, top_k, width, dropped, dtype):
    dtype = TYPES[dtype]
    ids = random_ids(n, n, top_k, 6, dropped)
    plan = M.expert_plan(ids, 6)
    off, order, pos = R.plan(ids.cpu().numpy(), 6)
    y, g = normal(1, n * top_k, width, dtype=dtype), normal(2, n, width, dtype=dtype)
    y[off[-1]:] = float("nan")                                   # rows that no expert owns are not read
    wt = normal(3, n, top_k)
    clean = f64(y)
    clean[off[-1]:] = 0
    for weights in (wt, None):
        w64 = None if weights is None else f64(weights)
        want = R.combine(clean, pos, w64)
        mag = R.combine(np.abs(clean), pos, None if weights is None else np.abs(w64))
        got = f64(M.expert_combine(y, plan, weights))
        # one fused multiply-add a slot
        assert np.all(np.abs(got - want) <= half_step(dtype) * np.abs(want) + 2 * top_k * U32 * mag + least(dtype))
        dy, dw = M.expert_combine_grad(g, y, plan, weights)
        want_y, want_w = R.combine_grad(f64(g), clean, pos, w64)
        assert np.all(np.abs(f64(dy) - want_y) <= (half_step(dtype) + 2 * U32) * np.abs(want_y) + least(dtype))
        _, mag_w = R.combine_grad(np.abs(f64(g)), np.abs(clean), pos, w64)
        # FP32 sums over the width
        assert np.all(np.abs(f64(dw) - want_w) <= (width + 16) * U32 * mag_w)
        only, none = M.expert_combine_grad(g, None, plan, weights)
        assert none is None and torch.equal(only, dy)


def test_combine_strides():
    n, top_k, width = 30, 3, 40
    ids = random_ids(1, n, top_k, 4, 0.2)
    plan = M.expert_plan(ids, 4)
    y = normal(1, n * top_k, width, dtype=torch.bfloat16)
    g = normal(2, n, width, dtype=torch.bfloat16)
    wt = normal(3, n, top_k)
    want, (wy, ww) = M.expert_combine(y, plan, wt), M.expert_combine_grad(g, y, plan, wt)
    for pad in (1, 8):
        big_y = torch.full((n * top_k, width + pad), 7.0, dtype=torch.bfloat16, device="cuda")
        big_g, out = big_y[:n].clone(), big_y[:n].clone()
        dy = big_y.clone()
        big_y[:, :width], big_g[:, :width] = y, g
        assert torch.equal(M.expert_combine(big_y[:, :width], plan, wt, out=out[:, :width]), want)
        a, b = M.expert_combine_grad(big_g[:, :width], big_y[:, :width], plan, wt, out=dy[:, :width])
        # the same FP32 products summed over the width in another order
        _, mag = R.combine_grad(np.abs(f64(g)), np.abs(f64(y)), plan.pos.cpu().numpy(), None)
        assert torch.equal(a, wy) and np.all(np.abs(f64(b) - f64(ww)) <= 2 * (width + 16) * U32 * mag)
        assert torch.all(out[:, width:] == 7) and torch.all(dy[:, width:] == 7)


# --------------------------------------------------- the run of them, as used --

def layer(x, gate, w1, w2, top_k, bias):
    """x -> route -> plan -> up product -> SiLU -> down product -> combine."""
    logits = x.float() @ gate.t()
    ids, weights = M.route(logits, top_k, score="sigmoid", bias=bias, groups=4, top_groups=2, group_score="top2")
    plan = M.expert_plan(ids, gate.shape[0])
    up = M.expert_gemm(x, w1, plan)
    act = torch.nn.functional.silu(up.float()).to(x.dtype)
    down = M.expert_gemm(act, w2, plan, gather=False)
    return logits, ids, weights, plan, up, act, down, M.expert_combine(down, plan, weights)


def layer_grad(go, x, gate, w1, w2, top_k, fwd):
    logits, ids, weights, plan, up, act, down, _ = fwd
    gdown, gweights = M.expert_combine_grad(go, down, plan, weights)
    gw2 = M.expert_gemm_grad_w(gdown, act, plan, gather=False)
    gact = M.expert_gemm_grad_x(gdown, w2, plan).float()
    s = torch.sigmoid(up.float())
    gup = (gact * s * (1 + up.float() * (1 - s))).to(x.dtype)
    gw1 = M.expert_gemm_grad_w(gup, x, plan)
    gx = M.expert_combine(M.expert_gemm_grad_x(gup, w1, plan), plan)
    glogits = M.route_grad(gweights, logits, ids, score="sigmoid")
    return gx.float() + glogits @ gate, glogits.t() @ x.float(), gw1, gw2


def layer_plain(x, gate, w1, w2, ids):
    """The layer in FP64 with its choice given, a loop over experts."""
    s = torch.sigmoid(x @ gate.t())
    w = s.gather(1, ids)
    w = w / w.sum(1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(gate.shape[0]):
        t, slot = (ids == e).nonzero(as_tuple=True)
        h = torch.nn.functional.silu(x[t] @ w1[e].t()) @ w2[e].t()
        out = out.index_add(0, t, w[t, slot, None] * h)
    return out


@pytest.mark.parametrize("n,top_k", [(1, 2), (190, 3)])
def test_layer_forward_and_gradients(n, top_k):
    experts, d, hidden = 16, 128, 192
    x = normal(1, n, d, dtype=torch.float16)
    gate = normal(2, experts, d, scale=d ** -0.5)
    w1 = normal(3, experts, hidden, d, dtype=torch.float16, scale=d ** -0.5)
    w2 = normal(4, experts, d, hidden, dtype=torch.float16, scale=hidden ** -0.5)
    bias = normal(5, experts, scale=0.05)
    go = normal(6, n, d, dtype=torch.float16)
    fwd = layer(x, gate, w1, w2, top_k, bias)
    grads = layer_grad(go, x, gate, w1, w2, top_k, fwd)
    leaves = [t.double().cpu().requires_grad_(True) for t in (x, gate, w1, w2)]
    want = layer_plain(*leaves, fwd[1].long().cpu())
    want.backward(go.double().cpu())
    # three FP16 roundings between input and output, each at most 2^-11 of a value of the scale of the result's
    # terms; gradients pass five.  Norm-wise that is under 5 * 2^-11 * sqrt(top_k); 0.01 leaves a factor of two.
    def off(a, b):
        return float(torch.linalg.vector_norm(a.double().cpu() - b) / torch.linalg.vector_norm(b))
    assert off(fwd[-1], want.detach()) < 0.005
    for got, leaf in zip(grads, leaves):
        assert off(got, leaf.grad) < 0.01


@pytest.mark.parametrize("n", [4, 40, 900])
def test_layer_captured_and_replayed(n):
    """The run captured once and replayed on other inputs equals the eager run, bit for bit, beside a second graph."""
    experts, d, hidden, top_k = 16, 128, 192, 3
    gate = normal(2, experts, d, scale=d ** -0.5)
    w1 = normal(3, experts, hidden, d, dtype=torch.bfloat16, scale=d ** -0.5)
    w2 = normal(4, experts, d, hidden, dtype=torch.bfloat16, scale=hidden ** -0.5)
    bias = normal(5, experts, scale=0.05)

    def whole(x, go):
        fwd = layer(x, gate, w1, w2, top_k, bias)
        return (fwd[-1], *layer_grad(go, x, gate, w1, w2, top_k, fwd))

    graphs = []
    for i in range(2):
        x, go = normal(20 + i, n, d, dtype=torch.bfloat16), normal(30 + i, n, d, dtype=torch.bfloat16)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            whole(x, go)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = whole(x, go)
        graphs.append((graph, x, go, outs))
    for seed in (40, 41):
        for i, (graph, x, go, outs) in enumerate(graphs):
            x.copy_(normal(seed + i, n, d, dtype=torch.bfloat16))
            go.copy_(normal(seed + 7 + i, n, d, dtype=torch.bfloat16))
        for graph, *_ in graphs:
            graph.replay()
        for graph, x, go, outs in graphs:
            for a, b in zip(outs, whole(x, go)):
                assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Rows and matrices that start more than 2^31 elements into their buffers: the last ones are checked."""
    dtype, n, top_k, width = torch.bfloat16, 300000, 4, 2048
    ids = torch.arange(n * top_k, dtype=torch.int32, device="cuda").view(n, top_k) % 3
    plan = M.expert_plan(ids, 3)
    y = torch.empty(n * top_k, width, dtype=dtype, device="cuda")
    assert y.numel() > 2 ** 31
    y.copy_((torch.arange(n * top_k, device="cuda") % 251)[:, None].to(dtype).expand(-1, width))
    out = M.expert_combine(y, plan)
    want = y[plan.pos.long().flatten(), 0].view(n, top_k).float().sum(1)       # sums of four integers under 251
    assert torch.equal(out[:, 0].float(), want.to(dtype).float()) and torch.equal(out[:, -1], out[:, 0])
    dy, dw = M.expert_combine_grad(out, y, plan)
    token = plan.order.long() // top_k
    assert torch.equal(dy[:, 5], out[token, 5]) and torch.equal(dy[-1], out[token[-1]])
    del y, dy, dw, out
    experts, k = 70, 4096                                                      # matrices of 8192 x 4096
    w = torch.zeros(experts, 8192, k, dtype=dtype, device="cuda")
    assert w.numel() > 2 ** 31
    w[-1] = normal(1, 8192, k, dtype=dtype, scale=k ** -0.5)
    for rows in (5, 400, 20000):
        x = normal(2, rows, k, dtype=dtype)
        plan = M.expert_plan(torch.full((rows, 1), experts - 1, dtype=torch.int32, device="cuda"), experts)
        got = M.expert_gemm(x, w, plan)
        at = [0, rows // 2, rows - 1]
        want, mag = f64(x[at]) @ f64(w[-1]).T, np.abs(f64(x[at])) @ np.abs(f64(w[-1])).T
        assert np.all(np.abs(f64(got[at]) - want) <= product_tolerance(want, mag, k, dtype))
        g = normal(3, rows, 8192, dtype=dtype)
        got = M.expert_gemm_grad_x(g, w, plan)
        want, mag = f64(g[at]) @ f64(w[-1]), np.abs(f64(g[at])) @ np.abs(f64(w[-1]))
        assert np.all(np.abs(f64(got[at]) - want) <= product_tolerance(want, mag, 8192, dtype))
    dw = M.expert_gemm_grad_w(g[:400], x[:400], M.expert_plan(torch.full((400, 1), experts - 1, dtype=torch.int32, device="cuda"), experts), out=w)
    want, mag = f64(g[:400]).T @ f64(x[:400, :64]), np.abs(f64(g[:400])).T @ np.abs(f64(x[:400, :64]))
    assert np.all(np.abs(f64(dw[-1, :, :64]) - want) <= product_tolerance(want, mag, 400, dtype))
    assert not dw[:-1].any()


def test_two_streams_at_once():
    """Calls on two streams share nothing: results equal those of one at a time."""
    sets = []
    for i in range(2):
        ids = random_ids(i, 4000, 8, 64, 0.1, 1.0)
        x = normal(i + 3, 4000, 128, dtype=torch.float16)
        w = normal(i + 5, 64, 136, 128, dtype=torch.float16)
        sets.append((ids, x, w, torch.cuda.Stream()))

    def work(ids, x, w):
        plan = M.expert_plan(ids, 64)
        y = M.expert_gemm(x, w, plan)
        return plan.order, y, M.expert_combine(y, plan), M.expert_gemm_grad_w(y, x, plan)

    want = [work(*s[:3]) for s in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        got = []
        for ids, x, w, stream in sets:
            with torch.cuda.stream(stream):
                got.append(work(ids, x, w))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for u, v in zip(a, b):
            assert torch.equal(u, v)


def test_mirror_refuses_on_the_gpu():
    x = normal(1, 4, 8)
    with pytest.raises(M.MpkError):
        M.route(x, 9)
    with pytest.raises(M.MpkError):
        M.route(x, 0)
    with pytest.raises(ValueError):
        M.route(x.t(), 2)                                        # columns, not rows, are contiguous
    with pytest.raises(ValueError):
        M.route(x[:1].expand(4, 8), 2)                           # rows that overlap
    with pytest.raises(ValueError):
        M.route(x, 2, bias=torch.zeros(8))                       # bias on the CPU
    with pytest.raises(ValueError):
        M.route(x, 2, bias=torch.zeros(7, device="cuda"))
    plan = M.expert_plan(torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 3)
    w = normal(2, 3, 16, 8, dtype=torch.float16)
    with pytest.raises(ValueError):
        M.expert_gemm(x, w, plan)                                # FP32 rows
    with pytest.raises(ValueError):
        M.expert_gemm(x.half(), w.bfloat16(), plan)
    with pytest.raises(ValueError):
        M.expert_gemm(x.half(), w[:2], plan)
    with pytest.raises(ValueError):
        M.expert_gemm(x.half(), w.transpose(1, 2), plan)
    with pytest.raises(ValueError):
        M.expert_gemm(x.half(), w, plan, out=torch.empty(8, 15, dtype=torch.float16, device="cuda"))


@pytest.mark.parametrize("score,bias,row,top_k", [("sigmoid", 0.0, [18, 18, 18.125], 1), ("sigmoid", 0.0, [20, 20, 21], 1),
                                                  ("sigmoid", 0.0, [20, 20, 21], 2), ("sigmoid", 0.0, [20, 21, 21], 2),
                                                  ("softmax", 0.1, [10, -15, -15, -14.9375], 2)])
def test_route_ties_at_the_cut(score, bias, row, top_k):
    """The last slot and the first loser have the same logit and bias, and FP32 cannot tell another loser, or the slot
    before, from them: the higher logit is chosen."""
    x = torch.tensor([row, row[::-1], row], dtype=torch.float32, device="cuda")
    check_route(x, top_k, score=score, bias=torch.full((len(row),), bias, device="cuda"))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,top_k", [(5, 2), (64, 1), (64, 6), (256, 8), (256, 31), (1000, 7)])
def test_route_ties_at_the_cut_of_coarse_logits(experts, top_k, score, dtype):
    """Few distinct logits and equal biases: exact ties everywhere, between values that FP32 scores round to one
    another (sigmoids of 16 to 20; softmax values 1e-11 beside a bias of 0.1) but FP64 tells apart."""
    rng = np.random.default_rng(experts + top_k)
    x = rng.integers(0, 9, size=(40, experts)) / 2 + (16 if score == "sigmoid" else -16)
    x[20:] = np.where(rng.random((20, experts)) < 0.9, x[20:].min(), x[20:])     # most at the lowest value
    if score == "softmax":
        x[:, 0] = 10
    x = torch.from_numpy(x.astype(np.float32)).to(TYPES[dtype]).cuda()
    check_route(x, top_k, score=score, bias=torch.full((experts,), 0.1 if score == "softmax" else 0.0, device="cuda"))
    if experts % 4 == 0:
        check_route(x, min(top_k, experts // 2), score=score, bias=torch.full((experts,), 0.1, device="cuda"), groups=4,
                    top_groups=2, group_score="top2")
    # biases one step apart: what is near a tie at the cut may have another bias
    steps = torch.from_numpy((np.float32(0.1) + rng.integers(0, 3, experts) * np.float32(2.0 ** -27)).astype(np.float32)).cuda()
    check_route(x, top_k, score=score, bias=steps)


@pytest.mark.parametrize("experts", [256, 512, 1024])
def test_route_near_ties_of_wide_rows(experts):
    """Softmax rows whose sum is many roundings long, with biases that put pairs of choice values within one another's
    error bound: c of one expert is that of the next to 1e-8."""
    rng = np.random.default_rng(experts)
    for scale in (0.01, 2.0):
        x = (scale * rng.normal(size=(30, experts))).astype(np.float32)
        s = R.softmax(x.astype(np.float64)).mean(0)
        bias = (0.1 - s).astype(np.float32)                    # all c of an average row equal
        check_route(torch.from_numpy(x).cuda(), 8, bias=torch.from_numpy(bias).cuda())
        same = np.tile(x[:1], (30, 1)) + (rng.integers(-2, 3, x.shape) * 2.0 ** -22 * np.abs(x)).astype(np.float32)
        bias = (0.1 - R.softmax(x[:1].astype(np.float64))[0]).astype(np.float32)
        for top_k in (1, 8):
            check_route(torch.from_numpy(same).cuda(), top_k, bias=torch.from_numpy(bias).cuda())


def test_plans_of_two_threads():
    """Two host threads that plan at once with different numbers of experts: every call returns its plan."""
    import threading
    sets = [(random_ids(e, 2000, 3, e, 0.1), e) for e in (1024, 40)]
    want = [R.plan(ids.cpu().numpy(), e) for ids, e in sets]
    plans, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(400):
                    plans[i].append(M.expert_plan(*sets[i]))
        except Exception as e:                                 # handed to the test's own thread
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for got, w in zip(plans, want):
        for p in got:
            for a, b in zip((p.offsets, p.order, p.pos), w):
                assert np.array_equal(a.cpu().numpy(), b)


def test_plans_of_many_blocks_captured_and_replayed():
    """Two plans of several blocks in one graph with one scratch, replayed on other ids."""
    experts, n, top_k = 160, 20000, 2
    ids = [random_ids(i, n, top_k, experts, 0.1, 1.0) for i in range(2)]
    need = int(M.lib().mpkExpertPlanBytes(n, top_k, experts))
    assert need > 0
    work = torch.full((need // 4,), -1, dtype=torch.int32, device="cuda")
    outs = [[torch.empty(c, dtype=torch.int32, device="cuda") for c in (experts + 1, n * top_k, n * top_k)] for _ in ids]

    def both():
        stream = torch.cuda.current_stream().cuda_stream
        for i, o in zip(ids, outs):
            assert M.lib().mpkExpertPlan(stream, i.data_ptr(), n, top_k, experts, *(t.data_ptr() for t in o),
                                         work.data_ptr(), need) == M.MPK_OK

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for seed in range(10, 16):
        for j, i in enumerate(ids):
            i.copy_(random_ids(seed + 100 * j, n, top_k, experts, 0.1, 1.0))
        graph.replay()
        for i, o in zip(ids, outs):
            for a, b in zip(o, R.plan(i.cpu().numpy(), experts)):
                assert np.array_equal(a.cpu().numpy(), b.reshape(-1))


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("n,top_k,experts,k,width", [(1, 1, 1, 64, 72), (4, 2, 4, 72, 40), (8, 2, 1, 520, 64), (40, 2, 20, 136, 64),
                                                     (200, 2, 3, 136, 264), (300, 2, 20, 72, 64), (30, 2, 3, 37, 33)])
def test_products_of_entries_that_name_no_row(n, top_k, experts, k, width, pad):
    """Entries outside the rows inside an expert's segment count as rows of zeros, whichever kernel runs and whatever
    the scratch held; the token that no entry names is not read."""
    dtype = torch.bfloat16
    plan = M.expert_plan(random_ids(n, n, top_k, experts), experts)
    m = n * top_k
    order = plan.order.clone()
    none = torch.tensor([-1, m, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    bad = order < top_k                                          # those of token 0
    order[bad] = none[torch.arange(int(bad.sum()), device="cuda") % 4]
    x = torch.full((n, k + pad), float("nan"), dtype=dtype, device="cuda")[:, :k]
    x[1:] = normal(1, n - 1, k, dtype=dtype)
    w = normal(2, experts, width, k, dtype=dtype, scale=k ** -0.5)
    g = normal(3, m, width, dtype=dtype)
    off = plan.offsets.cpu().numpy()
    clean = f64(x)
    clean[0] = 0
    xs = R.gathered(clean, np.where(bad.cpu().numpy(), -1, order.cpu().numpy()), top_k)
    lib, stream = M.lib(), torch.cuda.current_stream().cuda_stream
    ldx = x.stride(0)

    def scratch(grad_w):
        need = int(lib.mpkExpertGemmBytes(grad_w, m, experts, k))
        work = torch.full((need // 2 + 8,), float("nan"), dtype=dtype, device="cuda")
        return work, work.data_ptr(), need

    y = torch.empty(m, width, dtype=dtype, device="cuda")
    work, address, need = scratch(0)
    assert lib.mpkExpertGemm(stream, 2, x.data_ptr(), ldx, w.data_ptr(), k, width * k, plan.offsets.data_ptr(),
                             order.data_ptr(), top_k, m, experts, width, k, y.data_ptr(), width, address, need) == M.MPK_OK
    want, mag = R.gemm(xs, f64(w), off), R.gemm(np.abs(xs), np.abs(f64(w)), off)
    assert np.all(np.abs(f64(y) - want) <= product_tolerance(want, mag, k, dtype))
    assert torch.all(y[bad] == 0)
    dw = torch.empty(experts, width, k, dtype=dtype, device="cuda")
    work, address, need = scratch(1)
    assert lib.mpkExpertGemmGradW(stream, 2, g.data_ptr(), width, x.data_ptr(), ldx, plan.offsets.data_ptr(),
                                  order.data_ptr(), top_k, m, experts, width, k, dw.data_ptr(), k, width * k, address,
                                  need) == M.MPK_OK
    want, mag = R.gemm_grad_w(f64(g), xs, off), R.gemm_grad_w(np.abs(f64(g)), np.abs(xs), off)
    most = int((off[1:] - off[:-1]).max())
    assert np.all(np.abs(f64(dw) - want) <= product_tolerance(want, mag, most, dtype))


def test_route_far_sigmoids_keep_their_ratios():
    """Chosen sigmoids below the FP32 range beside one that is not: e^x of the lower, over the sum."""
    x = torch.full((5, 8), -300.0, device="cuda")
    for t, (a, b, c) in enumerate([(-50, -95.5, -110), (-59.5, -88, -104), (-30, -87.5, -90), (-0.5, -70, -85), (0.5, -40, -80)]):
        x[t, 2], x[t, 5], x[t, 7] = a, b, c
    for k in (2, 3):
        check_route(x, k, score="sigmoid")
        check_route(x, k, score="sigmoid", bias=torch.linspace(0, 1, 8, device="cuda").square()[[0, 1, 7, 2, 3, 6, 4, 5]].contiguous())
    ids, _ = M.route(x, 3, score="sigmoid")
    for slot in (1, 2):                                        # the gradient of one small weight: w (1 - s) (1 - w) there
        g = torch.zeros(5, 3, device="cuda")
        g[:, slot] = 1.0
        want = R.route_grad(f64(g), f64(x), ids.cpu().numpy(), score="sigmoid")
        got = f64(M.route_grad(g, x, ids, score="sigmoid"))
        at = np.arange(5), ids[:, slot].cpu().numpy()
        # the weight as in weights_close with logits of up to 300, and three factors
        assert np.all(np.abs(got - want)[at] <= 900 * U32 * np.abs(want[at]) + 1e-37)


@pytest.mark.parametrize("experts,n,top_k,k,width", [(64, 1500, 2, 512, 1024), (8, 3000, 4, 1024, 512)])
def test_products_of_many_tiles_a_cluster(experts, n, top_k, k, width):
    """Every cluster takes over more tiles than it has places for their indices: right, and the same bit for bit in
    every call, whichever cluster took which."""
    dtype = torch.bfloat16
    s = setup_products(5, n, top_k, experts, k, width, dtype, True, 0.05, 1)
    check_products(*s, True, dtype)
    plan, _, x, _, w, g = s

    def run():
        return M.expert_gemm(x, w, plan), M.expert_gemm_grad_x(g, w, plan), M.expert_gemm_grad_w(g, x, plan)

    first = run()
    for _ in range(20):
        for a, b in zip(first, run()):
            assert torch.equal(a, b)


def test_calls_refuse_to_lose_a_gradient():
    """The calls record no gradient: an input that needs one is refused while torch records, and taken otherwise."""
    x = normal(1, 6, 8).requires_grad_(True)
    with pytest.raises(ValueError, match="no_grad"):
        M.route(x, 2)
    with torch.no_grad():
        ids, weights = M.route(x, 2)
    plan = M.expert_plan(ids, 8)
    half = normal(2, 6, 16, dtype=torch.float16)
    w = torch.nn.Parameter(normal(3, 8, 24, 16, dtype=torch.float16))
    y = normal(4, 12, 16).requires_grad_(True)
    for call in (lambda: M.expert_gemm(half, w, plan), lambda: M.expert_combine(y, plan, weights),
                 lambda: M.expert_combine(y.detach(), plan, weights.clone().requires_grad_(True)),
                 lambda: M.expert_gemm_grad_x(normal(5, 12, 24, dtype=torch.float16), w, plan),
                 lambda: M.route_grad(weights, x, ids)):
        with pytest.raises(ValueError, match="no_grad"):
            call()
        with torch.no_grad():
            call()
    assert torch.equal(M.expert_gemm(half, w.detach(), plan), M.expert_gemm(half, w.data, plan))


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("n,top_k,experts,k,width", [(2, 2, 5, 37, 19), (40, 2, 10, 101, 67), (200, 2, 20, 75, 133), (300, 2, 3, 197, 301)])
def test_products_odd_widths_in_aligned_rows(n, top_k, experts, k, width, gather):
    """Rows of any length that start on 16-byte boundaries: the tensor-core and few-rows kernels, whose last pieces of a
    row hold what lies behind it (NaN here)."""
    dtype = torch.float16
    plan, off, x, xs, w, g = setup_products(6, n, top_k, experts, k, width, dtype, gather, 0.1, 0.5)

    def aligned(t, value=float("nan")):
        big = torch.full((*t.shape[:-1], (t.shape[-1] + 7) // 8 * 8 + 8), value, dtype=dtype, device="cuda")
        view = big[..., :t.shape[-1]]
        view.copy_(t)
        return view

    outs = [aligned(torch.zeros(shape, dtype=dtype, device="cuda"), 7.0) for shape in
            ((n * top_k, width), (n * top_k, k), (experts, width, k))]
    check_products(plan, off, aligned(x), xs, aligned(w), aligned(g), gather, dtype, outs)
    for o in outs:
        whole = o._base
        o.fill_(7.0)
        assert torch.all(whole == 7.0)
