"""Scored routing against its definition in 64 bits: the choice exactly, weights and gradients within fp32's steps."""

import pytest
import torch

import quantaweave_amd as qa
from tests import mx_oracle as ref

pytestmark = pytest.mark.gpu
INF = float("inf")

# (experts, groups, top_groups, top_k)
RULES = [(1, 1, 1, 1), (8, 1, 1, 2), (12, 3, 2, 5), (16, 16, 3, 3), (64, 1, 1, 64), (64, 8, 4, 6), (100, 5, 2, 7),
         (184, 8, 3, 4), (256, 8, 4, 8), (512, 16, 5, 9), (1000, 10, 10, 33), (1024, 64, 1, 16), (1024, 1, 1, 8)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check(logits, rule, score, bias=None, group_score="top2", renormalize=True, scale=1.0):
    experts, groups, top_groups, k = rule
    got = qa.route_experts(logits.cuda(), k, score=score, bias=None if bias is None else bias.cuda(), groups=groups,
                           top_groups=top_groups, group_score=group_score, renormalize=renormalize, scale=scale)
    want = ref.route(logits.double(), k, score, None if bias is None else bias.double(), groups, top_groups,
                     group_score, renormalize, scale)
    index, weight, scores = (t.cpu() for t in got)
    assert index.dtype == torch.int32 and torch.equal(index.long(), want[0])
    for a, b, steps in ((scores, want[2], 1), (weight, want[1], k + 4)):  # 64-bit scores rounded; k additions, a division, a product
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        a, b = torch.nan_to_num(a.double()), torch.nan_to_num(b)
        assert ((a - b).abs() <= 1.01 * steps * ref.EPS24 * b.abs() + 2.0 ** -149 * max(1.0, abs(scale)) * steps).all()
    return got


@pytest.mark.parametrize("tokens", [1, 3, 130])
@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(tokens, rule, score):
    g = gen(tokens + rule[0])
    logits, bias = 2 * torch.randn(tokens, rule[0], generator=g), 0.1 * torch.randn(rule[0], generator=g)
    check(logits, rule, score, bias)
    check(logits, rule, score, None, "max", False, 2.5)


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_and_near_ties(rule, score):
    """Equal logits go to the lowest index; logits one step of fp32 apart, and scores
    that fp32 cannot tell apart, are chosen as 64 bits do."""
    g = gen(rule[0])
    e = rule[0]
    few = torch.randint(0, 3, (40, e), generator=g).float()
    step = torch.ones(40, e)
    step = torch.where(torch.rand(40, e, generator=g) < 0.5, torch.nextafter(step, 2 * step), step)
    high = 12 + torch.rand(40, e, generator=g)  # sigmoids within 2^-17 of 1
    for z in (few, step, high, torch.zeros(2, e)):
        check(z, rule, score)
        check(z, rule, score, 0.25 * torch.randint(0, 2, (e,), generator=g).float(), "max")


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_infinite_and_nan_rows(rule, score):
    g = gen(7 + rule[0])
    e = rule[0]
    z = torch.randn(9, e, generator=g)
    z[0] = -INF                                   # nothing left: scores and weights 0
    z[1, torch.rand(e, generator=g) < 0.7] = -INF
    z[2] = torch.finfo(torch.float32).min         # a mask of the type's lowest value
    z[3, : e // 2] = torch.finfo(torch.float32).min
    z[4, e // 2] = float("nan")
    z[5] = float("nan")
    z[6, 0] = INF if score == "sigmoid" else 80.0
    z[7] = -100.0                                 # every sigmoid 4e-44
    got = check(z, rule, score)
    assert not got[1][0].any() and not got[2][0].any()
    bias = torch.randn(e, generator=g)
    bias[torch.rand(e, generator=g) < 0.3] = -INF  # experts switched off
    check(z, rule, score, bias)
    bias[0] = float("nan")
    check(z, rule, score, bias, "max")


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient(rule, score, renormalize):
    g = gen(rule[0] * 3)
    e, groups, top_groups, k = rule
    t, scale = 21, 1.5
    z = torch.randn(t, e, generator=g)
    dw, ds = torch.randn(t, k, generator=g), torch.randn(t, e, generator=g)
    zc = z.cuda().requires_grad_(True)
    index, weight, scores = qa.route_experts(zc, k, score=score, groups=groups, top_groups=top_groups,
                                             renormalize=renormalize, scale=scale)
    zd = z.double().requires_grad_(True)
    want = ref.route(zd, k, score, None, groups, top_groups, "top2", renormalize, scale)
    assert torch.equal(index.cpu().long(), want[0])
    s = want[2].detach()
    picked = s.gather(1, want[0])
    total = picked.sum(1, keepdim=True) if renormalize else torch.ones(t, 1).double()
    for use_w, use_s in ((True, True), (True, False), (False, True)):
        outs = [o for o, u in ((weight, use_w), (scores, use_s)) if u]
        grads = [d for d, u in ((dw, use_w), (ds, use_s)) if u]
        (got,) = torch.autograd.grad(outs, zc, [d.cuda() for d in grads], retain_graph=True)
        (exact,) = torch.autograd.grad([o for o, u in ((want[1], use_w), (want[2], use_s)) if u], zd,
                                       [d.double() for d in grads], retain_graph=True)
        # the largest a term of ds can be; every sum has at most e + k + 16 roundings
        big = torch.zeros_like(s)
        if use_s:
            big += ds.double().abs()
        if use_w:
            part = scale * dw.double().abs()
            both = part + ((part * picked).sum(1, keepdim=True) / total if renormalize else 0.0)
            big.scatter_add_(1, want[0], both / total)
        bound = (e + k + 16) * ref.EPS24 * s * (big + (big * s).sum(1, keepdim=True)) + 1e-37
        assert ((got.cpu().double() - exact).abs() <= bound).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_against_differences(score):
    """Central differences of the definition in 64 bits along random directions."""
    g = gen(77)
    e, k = 48, 4
    z = torch.randn(6, e, generator=g)
    bias = 0.1 * torch.randn(e, generator=g)
    dw, ds, v = torch.randn(6, k, generator=g), torch.randn(6, e, generator=g), torch.randn(6, e, generator=g)
    zc = z.cuda().requires_grad_(True)
    index, weight, scores = qa.route_experts(zc, k, score=score, bias=bias.cuda(), groups=6, top_groups=3)
    (got,) = torch.autograd.grad((weight, scores), zc, (dw.cuda(), ds.cuda()))
    picked = index.cpu().long()

    def loss(u):  # the choice held, as the gradient holds it
        s = torch.sigmoid(u) if score == "sigmoid" else torch.softmax(u, 1)
        p = s.gather(1, picked)
        return ((p / (p.sum(1, keepdim=True) + 1e-20)) * dw.double()).sum() + (s * ds.double()).sum()

    h = 1e-5
    diff = (loss(z.double() + h * v.double()) - loss(z.double() - h * v.double())) / (2 * h)
    # the differences' own error is about h^2 and 1e-16 / h; the gradient's a few hundred fp32 steps of its terms
    assert abs(float(diff) - float((got.cpu().double() * v.double()).sum())) <= 1e-5 * float((got.cpu().abs() * v.abs()).sum() + 1)


def test_shapes_and_strides():
    g = gen(2)
    z = torch.randn(3, 5, 80, generator=g)
    for v in (z[..., :64], z.transpose(0, 1)[..., ::2], z[0, 0], z[:0], z[:1].expand(4, 5, 80)):
        e = v.size(-1)
        index, weight, scores = qa.route_experts(v.cuda(), 3, score="sigmoid", groups=4, top_groups=2)
        assert index.shape == weight.shape == (*v.shape[:-1], 3) and scores.shape == v.shape
        want = ref.route(v.reshape(-1, e).double(), 3, "sigmoid", None, 4, 2)
        assert torch.equal(index.cpu().reshape(-1, 3).long(), want[0])


def test_empty_batch_has_a_gradient():
    z = torch.empty(0, 16, device="cuda", requires_grad=True)
    _, weight, scores = qa.route_experts(z, 2)
    (gz,) = torch.autograd.grad((weight, scores), z, (torch.empty_like(weight), torch.empty_like(scores)))
    assert gz.shape == z.shape


def test_broadcast_gradients_add_up():
    """A row of logits shared by all tokens gets the sum of their gradients."""
    g = gen(4)
    z = torch.randn(1, 32, generator=g).cuda().requires_grad_(True)
    _, weight, _ = qa.route_experts(z.expand(7, 32), 4, score="sigmoid")
    dw = torch.randn(7, 4, generator=g).cuda()
    (gz,) = torch.autograd.grad(weight, z, dw)
    _, one, _ = qa.route_experts(z, 4, score="sigmoid")
    (g1,) = torch.autograd.grad(one, z, dw.sum(0, keepdim=True))
    assert torch.allclose(gz, g1, rtol=0, atol=64 * 2.0 ** -24 * float(dw.abs().sum()))


def test_refusals():
    z = torch.randn(4, 16).cuda()
    for kw, match in ((dict(score="relu"), "score"), (dict(groups=3), "divide"), (dict(groups=4, top_groups=5), "top_groups"),
                      (dict(groups=4, top_groups=0), "top_groups"), (dict(group_score="min"), "group_score"),
                      (dict(scale=INF), "scale"), (dict(bias=torch.zeros(15).cuda()), "bias"),
                      (dict(bias=torch.zeros(16)), "bias")):
        with pytest.raises(ValueError, match=match):
            qa.route_experts(z, 2, **kw)
    for k in (0, 17):
        with pytest.raises(ValueError, match="top_k"):
            qa.route_experts(z, k)
    with pytest.raises(ValueError, match="top_k"):
        qa.route_experts(z, 5, groups=4, top_groups=1)
    with pytest.raises(ValueError, match="float32"):
        qa.route_experts(z.bfloat16(), 2)
