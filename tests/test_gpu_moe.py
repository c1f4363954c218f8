"""The sparse MLP of a few tokens on the GPU against its 64-bit specification.

Tolerance, with u half a step of the type (bf16 2^-8, fp16 2^-11): y is rounded (u
|y|), h is rounded (u sum |w d h|, and in fp16 half a step of the smallest
subnormals, 2^-25 sum |w d|), sums of H and of I products in fp32 (n 2^-23 of the
absolute products each, rounded or cut), and 2^-20 for the router weights and the
exponentials of silu (some steps of fp32).

A weight e^z / sum e^z is off by 2^-21 of itself (exponentials, sum and division,
some steps of fp32) and by what its logits are: a lane adds H / 32 exact products in fp32,
so a logit is off by d <= H / 32 2^-24 sum |x r|, and the quotient by e^(2 d) - 1 <= 2.1 d."""
import numpy as np
import pytest
import torch

from oracle import decode_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def inputs(T, H, I, E, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    return [t.to(DT[dtype]) for t in (n(T, H), n(E, H) * 1.3 / H ** 0.5, n(E, 2 * I, H) / H ** 0.5, n(E, H, I) / I ** 0.5)]


def check(x, router, gu, down, k, norm=True, scale=1.0, **kw):
    from kvr_b200 import kernels as K
    y, ids, w = K.moe_layer(x, router, gu, down, k, norm_topk=norm, scale=scale, return_routing=True, **kw)
    K.moe_status()
    f = lambda t: t.double().cpu().numpy()  # noqa: E731
    wy, wi, ww, by_h, by_sums, by_one = R.moe(f(x), f(router), f(gu), f(down), k, norm, scale)
    assert np.array_equal(ids.cpu().numpy(), wi)
    d = -(-x.shape[1] // 256) * 8 * 2.0 ** -24 * (np.abs(f(x)) @ np.abs(f(router)).T).max(1, keepdims=True)
    assert (np.abs(f(w) - ww) <= (2.0 ** -21 + 2.1 * d) * ww).all()
    u = torch.finfo(x.dtype).eps / 2
    H, I = x.shape[1], down.shape[2]
    tol = (u + 2.0 ** -20) * np.abs(wy) + (u + 2.0 ** -20 + 2.1 * d + I * 2.0 ** -23) * (1 + u) * by_h + H * 2.0 ** -23 * by_sums + 2.0 ** -25 * by_one
    err = np.abs(f(y) - wy)
    assert (err <= tol).all(), (err / tol).max()
    assert y.dtype is x.dtype
    return y


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,H,I,E,k", [
    (1, 64, 16, 1, 1), (1, 8, 8, 3, 2), (2, 72, 40, 5, 3), (1, 1024, 512, 16, 2), (5, 512, 264, 60, 5), (17, 256, 104, 128, 8),
    (64, 200, 136, 9, 9), (128, 128, 64, 4, 2), (128, 328, 72, 130, 8), (33, 1544, 1000, 12, 4), (128, 64, 32, 512, 16),
    (16, 64, 2048, 2, 1), (100, 136, 24, 300, 1)])
def test_layer(T, H, I, E, k, dtype):
    check(*inputs(T, H, I, E, dtype, T + H), k)


@pytest.mark.parametrize("norm,scale", [(False, 1.0), (True, 2.5), (False, 0.5)])
def test_weights(norm, scale):
    check(*inputs(9, 256, 96, 24, "bf16", 3), 4, norm, scale)


@pytest.mark.parametrize("T,H,I,E,k", [(128, 1096, 520, 2, 2), (65, 520, 1032, 3, 3), (128, 2056, 72, 1, 1), (48, 1160, 776, 2, 1),
                                       (96, 72, 1544, 4, 3), (112, 648, 392, 6, 5), (32, 2056, 1288, 8, 2)])
def test_many_tokens_an_expert(T, H, I, E, k):
    """Stages of every size, many rounds of the ring in both products, widths that end inside a block."""
    check(*inputs(T, H, I, E, "bf16", T + I), k)


def test_rows_far_apart():
    """Rows of x whose places pass 32 bits in bytes."""
    x, router, gu, down = inputs(128, 136, 72, 5, "bf16", 4)
    far = torch.empty(127 * (1 << 24) + 136, dtype=x.dtype, device=DEV).as_strided((128, 136), (1 << 24, 1))
    far.copy_(x)
    check(far, router, gu, down, 2)


def test_every_token_to_the_same_experts():
    """128 tokens on two experts of 64: segments of many columns, most experts without any."""
    x, router, gu, down = inputs(128, 256, 96, 64, "bf16", 5)
    x[:, 0], router[:, 0] = 1.0, 0.0
    router[7, 0] = router[40, 0] = 30.0
    check(x, router, gu, down, 2)


def test_equal_logits_go_to_the_lowest_experts():
    x, router, gu, down = inputs(6, 128, 64, 20, "f16", 6)
    router[:] = router[:1]
    check(x, router, gu, down, 3)


def test_strided_inputs():
    x, router, gu, down = inputs(10, 256, 96, 8, "bf16", 7)
    wide = torch.zeros(10, 512, dtype=x.dtype, device=DEV)
    wide[:, 64:320] = x
    gu2 = torch.zeros(8, 200, 264, dtype=x.dtype, device=DEV)
    gu2[:, :192, :256] = gu
    d2 = torch.zeros(8, 260, 104, dtype=x.dtype, device=DEV)
    d2[:, :256, :96] = down
    a = check(wide[:, 64:320], router, gu2[:, :192, :256], d2[:, :256, :96], 3)
    b = check(x, router, gu, down, 3)
    assert torch.equal(a, b)
    odd = torch.zeros(10, 259, dtype=x.dtype, device=DEV)  # rows that TMA cannot read are copied
    odd[:, 3:] = x
    assert torch.equal(check(odd[:, 3:], router, gu, down, 3), b)


def test_a_bad_token_stays_alone():
    from kvr_b200 import kernels as K
    x, router, gu, down = inputs(40, 256, 96, 8, "bf16", 8)
    good, ids, w = K.moe_layer(x, router, gu, down, 2, return_routing=True)
    x[3, 17], x[20, 5], x[39, 0] = float("nan"), float("inf"), -float("inf")
    y, ids2, w2 = K.moe_layer(x, router, gu, down, 2, return_routing=True)
    K.moe_status()
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 20, 39]] = True
    assert y[bad].isnan().all() and w2[bad].isnan().all() and ((ids2 >= 0) & (ids2 < 8)).all()
    assert torch.equal(y[~bad], good[~bad]) and torch.equal(ids2[~bad], ids[~bad])


def test_repeats_and_no_tokens():
    from kvr_b200 import kernels as K
    a = inputs(77, 512, 200, 40, "bf16", 9)
    first = K.moe_layer(*a, 6)
    for _ in range(20):
        assert torch.equal(K.moe_layer(*a, 6), first)
    y, ids, w = K.moe_layer(a[0][:0], *a[1:], 6, return_routing=True)
    assert y.shape == (0, 512) and ids.shape == (0, 6) and w.shape == (0, 6)
    K.moe_status()


def test_graph_and_streams():
    """A captured call replayed with new inputs, beside calls on two other streams."""
    from kvr_b200 import kernels as K
    x, router, gu, down = inputs(24, 512, 200, 32, "f16", 10)
    K.moe_status()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = K.moe_layer(x, router, gu, down, 4)
    others = [inputs(t, 512, 200, 32, "f16", 10 + t) for t in (1, 128)]
    want = [K.moe_layer(*o, 4) for o in others]
    streams = [torch.cuda.Stream() for _ in others]
    for seed in (1, 2, 3):
        new = inputs(24, 512, 200, 32, "f16", seed)
        for a, b in zip((x, router, gu, down), new):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        got = []
        for s, o in zip(streams, others):
            with torch.cuda.stream(s):
                got += [K.moe_layer(*o, 4) for _ in range(5)]
        torch.cuda.synchronize()
        assert torch.equal(y, K.moe_layer(*new, 4))
        assert all(torch.equal(g, want[i // 5]) for i, g in enumerate(got))
    K.moe_status()


def test_a_wait_that_ran_out_is_reported():
    """The status word that the waits set, set by the self-test's wait: reported once, then calls go on."""
    from kvr_b200 import _native as N
    from kvr_b200 import kernels as K
    a = inputs(3, 64, 16, 4, "f16", 11)
    want = K.moe_layer(*a, 2)
    K.moe_status()
    N.call("kvr_selftest_bounded_wait", K._moe_status(a[0].device).data_ptr(), 1000, N.stream())
    with pytest.raises(N.KvrError, match="gave up"):
        K.moe_status()
    K.moe_status()
    assert torch.equal(K.moe_layer(*a, 2), want)


# ------------------------------------------------ h, in two parts of the type --


def paired(T, H, I, E, dtype, seed, big=1.0):
    """Inner channels in pairs: nearly the same h, opposite columns of down.  y is small against sum |w d h|, so that what h
    loses on its way shows; positive x, gate and up keep the absolute products near the products."""
    dt = DT[dtype]
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    gate, up = (0.2 + r(E, I // 2, H)) / H ** 0.5, big * (0.2 + r(E, I // 2, H)) / H ** 0.5
    gate, up = (t.repeat_interleave(2, 1).to(dt) for t in (gate, up))
    other = 1 + torch.finfo(dt).eps * torch.randint(1, 3, (E, I // 2, H), generator=g)  # a step or two of the type
    up[:, 1::2] = (up[:, 1::2].float() * other).to(dt)
    down = (torch.randn(E, H, I // 2, generator=g) / I ** 0.5).repeat_interleave(2, 2).to(dt)
    down[:, :, 1::2] *= -1
    # (a router of zeros: every expert has the weight 1 / E, exactly)
    return [t.to(DEV) for t in ((0.25 + r(T, H)).to(dt), torch.zeros(E, H, dtype=dt), torch.cat([gate, up], 1), down)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,H,I,E", [(1, 16, 16, 1), (16, 16, 16, 1), (40, 24, 16, 1), (128, 16, 24, 1), (128, 64, 128, 1), (9, 16, 16, 4),
                                     (70, 32, 200, 2)])
def test_h_keeps_what_one_rounding_drops(T, H, I, E, dtype):
    """The bar of the tests above, with h rounded twice in place of once: h in two parts of the type is off by u^2 |h|, and
    in fp16, whose smallest step is 2^-24, by half of that at least.  (Weights of 1 / E: no error of the router.)"""
    from kvr_b200 import kernels as K
    x, router, gu, down = paired(T, H, I, E, dtype, T + H)
    f = lambda t: t.double().cpu().numpy()  # noqa: E731
    wy, _, _, by_h, by_sums, by_one = R.moe(f(x), f(router), f(gu), f(down), E)
    u = torch.finfo(x.dtype).eps / 2
    tol = (u + 2.0 ** -20) * np.abs(wy) + (u * u + 2.0 ** -20 + I * 2.0 ** -23) * (1 + u) * by_h + H * 2.0 ** -23 * by_sums
    tol += 2.0 ** -25 * by_one if dtype == "f16" else 0.0
    # (the bar tells: h rounded once, and all else exact, does not pass it)
    z = np.einsum("eih,th->tei", f(gu), f(x))
    h = z[..., :I] / (1 + np.exp(-z[..., :I])) * z[..., I:]
    once = np.einsum("tei,ehi->th", torch.tensor(h).to(x.dtype).double().numpy(), f(down)) / E
    assert (np.abs(once - wy) > tol).any()
    y = f(K.moe_layer(x, router, gu, down, E))
    K.moe_status()
    assert (np.abs(y - wy) <= tol).all(), (np.abs(y - wy) / tol).max()


def test_h_above_the_largest_half():
    """fp16: an h of up to twice the type's largest value is its largest value and a rest, off by half a step of the rest."""
    from kvr_b200 import kernels as K
    x, router, gu, down = paired(30, 16, 16, 1, "f16", 3, big=14000.0)
    down = (torch.randn(1, 16, 16, generator=torch.Generator().manual_seed(4)) / 256).half().to(DEV)
    f = lambda t: t.double().cpu().numpy()  # noqa: E731
    wy, _, _, by_h, by_sums, by_one = R.moe(f(x), f(router), f(gu), f(down), 1)
    z = f(x) @ f(gu)[0].T
    h = z[:, :16] / (1 + np.exp(-z[:, :16])) * z[:, 16:]
    assert (h > 65504).mean() > 0.2 and h.max() < 131008 and np.abs(wy).max() < 65504
    u = 2.0 ** -11
    rest = np.maximum(u * h, h - 65504)  # at most
    d = np.abs(f(down)[0])
    tol = (u + 2.0 ** -20) * np.abs(wy) + (2.0 ** -20 + 16 * 2.0 ** -23) * (1 + u) * by_h + (u * rest) @ d.T + 16 * 2.0 ** -23 * by_sums
    tol += 2.0 ** -25 * by_one
    assert (np.abs(np.minimum(h, 65504) @ f(down)[0].T - wy) > tol).any()  # (the bar tells)
    y = f(K.moe_layer(x, router, gu, down, 1))
    K.moe_status()
    assert (np.abs(y - wy) <= tol).all(), (np.abs(y - wy) / tol).max()


@pytest.mark.parametrize("T,H,I,E,k", [(1, 65536, 8, 2, 1), (70, 65536, 16, 3, 2), (2, 8, 131072, 2, 2), (128, 8, 8, 512, 16), (128, 40, 24, 16, 16),
                                       (3, 32768, 64, 4, 4), (1, 24, 1048576, 1, 1), (128, 104, 56, 1, 1)])
def test_the_largest_and_the_smallest_sizes(T, H, I, E, k):
    check(*inputs(T, H, I, E, "bf16", T + H), k)
