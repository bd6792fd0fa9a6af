"""Routing operators (include/mpkexperts.h) without a GPU: what the entry points refuse before they touch the
device, and the FP64 definitions of tests/experts_ref.py against finite differences."""
import ctypes

import numpy as np
import pytest

import experts_ref as R

torch = pytest.importorskip("torch")
import mpkmeans_b200 as M  # noqa: E402

INVALID = M.MPK_ERR_INVALID
FAKE = 4096                     # an address that no refused call may read


def params(**kw):
    p = M.mpkRouteParams()
    M.lib().mpkRouteParamsInit(ctypes.byref(p))
    p.experts, p.top_k = 16, 2
    for k, v in kw.items():
        setattr(p, k, v)
    return ctypes.byref(p)


def test_route_defaults():
    p = M.mpkRouteParams()
    M.lib().mpkRouteParamsInit(ctypes.byref(p))
    assert (p.experts, p.top_k, p.score, p.groups, p.top_groups, p.group_score, p.renormalize, p.scale) == \
        (0, 0, 0, 1, 1, 0, 1, 1.0)


@pytest.mark.parametrize("bad", [dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=17), dict(experts=64, top_k=33),
                                 dict(score=2), dict(score=-1), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(groups=0), dict(groups=3), dict(experts=66, groups=33), dict(groups=4, top_groups=5),
                                 dict(groups=4, top_groups=0), dict(group_score=2)])
def test_route_refuses_params(bad):
    assert M.lib().mpkRoute(None, params(**bad), FAKE, 0, 4, 2000, None, FAKE, FAKE) == INVALID
    if not set(bad) & {"groups", "top_groups", "group_score"}:
        assert M.lib().mpkRouteGrad(None, params(**bad), FAKE, 0, 4, 2000, FAKE, FAKE, FAKE, 2000) == INVALID


def test_route_refuses_arguments():
    lib = M.lib()
    good = [None, params(), FAKE, 0, 4, 16, None, FAKE, FAKE]
    for at, value in ((1, None), (2, None), (3, 3), (3, -1), (4, -1), (5, 15), (7, None), (8, None)):
        args = list(good)
        args[at] = value
        assert lib.mpkRoute(*args) == INVALID, (at, value)
    good = [None, params(), FAKE, 0, 4, 16, FAKE, FAKE, FAKE, 16]
    for at, value in ((1, None), (2, None), (3, 3), (4, -1), (5, 15), (6, None), (7, None), (8, None), (9, 15)):
        args = list(good)
        args[at] = value
        assert lib.mpkRouteGrad(*args) == INVALID, (at, value)
    assert lib.mpkRoute(None, params(), None, 0, 0, 16, None, None, None) == M.MPK_OK
    assert lib.mpkRouteGrad(None, params(), None, 0, 0, 16, None, None, None, 16) == M.MPK_OK


def test_plan_refuses():
    lib = M.lib()
    for n, k, e in ((-1, 2, 4), (4, 0, 4), (4, 2, 0), (4, 2, 1025), (1 << 29, 4, 4)):
        assert lib.mpkExpertPlan(None, FAKE, n, k, e, FAKE, FAKE, FAKE, None, 0) == INVALID
    for missing in (1, 5, 6, 7):
        args = [None, FAKE, 4, 2, 4, FAKE, FAKE, FAKE, None, 0]
        args[missing] = None
        assert lib.mpkExpertPlan(*args) == INVALID
    need = lib.mpkExpertPlanBytes(1 << 20, 8, 64)
    assert need > 0 and lib.mpkExpertPlanBytes(100, 8, 64) == 0
    assert lib.mpkExpertPlan(None, FAKE, 1 << 20, 8, 64, FAKE, FAKE, FAKE, FAKE, need - 1) == INVALID
    assert lib.mpkExpertPlan(None, FAKE, 1 << 20, 8, 64, FAKE, FAKE, FAKE, None, need) == INVALID
    assert lib.mpkExpertPlan(None, FAKE, 1 << 20, 8, 64, FAKE, FAKE, FAKE, FAKE + 2, need) == INVALID


def refused(fn, good, changes):
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert getattr(M.lib(), fn)(*args) == INVALID, (fn, at, value)


def test_products_refuse():
    # stream, type, X, ldx, W, ldw, strideW, offsets, order, top_k, m, experts, width, k, Y, ldy, work, bytes
    refused("mpkExpertGemm", [None, 2, FAKE, 64, FAKE, 64, 64 * 32, FAKE, FAKE, 2, 800, 4, 32, 64, FAKE, 32, FAKE, 1 << 30],
            [(1, 0), (1, 3), (2, None), (3, 63), (4, None), (5, 63), (6, 64 * 32 - 1), (7, None), (9, 0), (9, 3),
             (10, -1), (10, 1 << 30), (11, 0), (11, 1025), (12, 0), (12, (1 << 20) + 1), (13, 0), (14, None), (15, 31), (16, None), (16, 4104), (17, 800 * 64 * 2 - 1)])
    # stream, type, GY, ldgy, W, ldw, strideW, offsets, m, experts, width, k, GX, ldgx
    refused("mpkExpertGemmGradX", [None, 1, FAKE, 32, FAKE, 64, 64 * 32, FAKE, 8, 4, 32, 64, FAKE, 64],
            [(1, 0), (2, None), (3, 31), (4, None), (5, 63), (6, 64 * 32 - 1), (7, None), (8, -1), (9, 0), (10, 0),
             (11, 0), (12, None), (13, 63)])
    # stream, type, GY, ldgy, X, ldx, offsets, order, top_k, m, experts, width, k, GW, ldw, strideW, work, bytes
    refused("mpkExpertGemmGradW", [None, 1, FAKE, 32, FAKE, 64, FAKE, FAKE, 2, 8, 4, 32, 64, FAKE, 64, 64 * 32, FAKE, 1 << 30],
            [(1, 0), (2, None), (3, 31), (4, None), (5, 63), (6, None), (8, 0), (8, 3), (9, -1), (10, 0), (11, 0),
             (12, 0), (13, None), (14, 63), (15, 64 * 32 - 1), (16, None), (16, 4104), (17, 8 * 64 * 2 - 1)])
    assert M.lib().mpkExpertGemmBytes(0, 8, 4, 64) == 0 and M.lib().mpkExpertGemmBytes(0, 800, 4, 64) == 800 * 64 * 2


def test_combine_refuses():
    # stream, type, Y, ldy, pos, weights, n, top_k, width, out, ldo
    refused("mpkExpertCombine", [None, 0, FAKE, 8, FAKE, FAKE, 4, 2, 8, FAKE, 8],
            [(1, 3), (2, None), (3, 7), (4, None), (6, -1), (6, 1 << 30), (7, 0), (7, 1025), (8, 0), (9, None), (10, 7)])
    # stream, type, GO, ldgo, Y, ldy, pos, rows, weights, n, top_k, width, GY, ldgy, GW
    refused("mpkExpertCombineGrad", [None, 0, FAKE, 8, FAKE, 8, FAKE, FAKE, FAKE, 4, 2, 8, FAKE, 8, FAKE],
            [(1, 3), (2, None), (3, 7), (4, None), (5, 7), (6, None), (7, None), (9, -1), (10, 0), (11, 0), (12, None),
             (13, 7)])


def test_mirror_refuses_tensors():
    ids = torch.zeros(4, 2, dtype=torch.int32)
    plan = object.__new__(M.ExpertPlan)
    plan.n, plan.top_k, plan.rows, plan.experts = 4, 2, 8, 3
    plan.offsets = plan.order = plan.pos = ids
    for call in (lambda: M.route(torch.zeros(4, 8), 2),                                # not on the GPU
                 lambda: M.route(torch.zeros(8), 2),
                 lambda: M.route(torch.zeros(4, 8, dtype=torch.float64), 2),
                 lambda: M.route_grad(torch.zeros(4, 2), torch.zeros(4, 8), ids[0]),
                 lambda: M.expert_plan(ids, 3),
                 lambda: M.expert_plan(ids[0], 3),
                 lambda: M.expert_plan(ids.long(), 3),
                 lambda: M.ExpertPlan(torch.zeros(4, dtype=torch.int32), torch.zeros(7, dtype=torch.int32), ids),
                 lambda: M.ExpertPlan(torch.zeros(1, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), ids),
                 lambda: M.expert_gemm(torch.zeros(4, 8), torch.zeros(3, 8, 8), plan),   # FP32
                 lambda: M.expert_gemm(torch.zeros(5, 8, dtype=torch.half), torch.zeros(3, 8, 8, dtype=torch.half), plan),
                 lambda: M.expert_gemm_grad_x(torch.zeros(8, 8, dtype=torch.half), torch.zeros(3, 8, 8), plan),
                 lambda: M.expert_gemm_grad_w(torch.zeros(8, 8, dtype=torch.half), torch.zeros(4, 8, dtype=torch.bfloat16), plan),
                 lambda: M.expert_combine(torch.zeros(7, 8), plan),
                 lambda: M.expert_combine_grad(torch.zeros(4, 8), torch.zeros(8, 8), plan)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        M._route_params(8, 2, "tanh", 1, 1, "max", True, 1.0)
    with pytest.raises(ValueError):
        M._route_params(8, 2, "softmax", 1, 1, "mean", True, 1.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_reference_gradient_against_differences(score, renormalize):
    rng = np.random.default_rng(3)
    x = rng.normal(size=(5, 9))
    x[1, 2] = -np.inf
    ids, _ = R.route(x, 3, score=score)
    g = rng.normal(size=(5, 3))

    def loss(y):
        s = R.scores(y, score)
        w = np.take_along_axis(s, ids.astype(np.int64), 1)
        if renormalize:
            w = w / w.sum(1, keepdims=True)
        return (w * g * 1.5).sum()

    want = R.route_grad(g, x, ids, score=score, renormalize=renormalize, scale=1.5)
    h = 1e-5
    for t in range(5):
        for j in range(9):
            if np.isinf(x[t, j]):
                assert want[t, j] == 0
                continue
            up, down = x.copy(), x.copy()
            up[t, j] += h
            down[t, j] -= h
            # central differences: error h^2 / 6 times a third derivative of order one
            assert abs((loss(up) - loss(down)) / (2 * h) - want[t, j]) < 1e-8


def test_mirror_refuses_to_lose_a_gradient():
    """While torch records, a tensor that needs a gradient is refused before anything is called."""
    M._types()
    with pytest.raises(ValueError, match="no_grad"):
        M._run("mpkRoute", (torch.zeros(2), torch.zeros(2, requires_grad=True)))
