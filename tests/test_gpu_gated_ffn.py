"""aitk_gated_ffn_fwd / _bwd (both projections, activation and product in one launch; dx and the weight gradients in one launch) on the MI355X against 64-bit formulas: ragged
and tiny sizes around every tile border, both tile sizes, fused and separate weights, biases, frozen weights, pitches, determinism, another stream, replayed graphs.

Bounds, per element, u = 2^-8 (half a bf16 step): products of K terms in fp32 are off by at most c = 2^-14 of the terms' absolute values.  h is rounded once; the saved
value and gate once; du, dz are formed from the saved ones (|act'| < 1.2, |act''| < 1.2) and rounded once; every gradient is rounded once.  In the 2-norm these at most four
roundings, each below u of its value and stretched by at most 1.2, stay below 6 u of the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
U, FP = 2.0 ** -8, 2.0 ** -14


def _act(z, act):
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        c = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    k0, k1 = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(k0 * (z + k1 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k0 * (1 + 3 * k1 * z * z)


def _want(x, wv, wg, bv, bg, dh, act):
    x, wv, wg, dh = x.double(), wv.double(), wg.double(), dh.double()
    bv, bg = (0.0 if b is None else b.double() for b in (bv, bg))
    wvt, wgt = wv.t().contiguous(), wg.t().contiguous()
    u, z = x @ wvt + bv, x @ wgt + bg
    eu, ez = FP * (x.abs() @ wvt.abs() + abs(bv)), FP * (x.abs() @ wgt.abs() + abs(bg))
    f, s = _act(z, act)
    h = u * f
    r = {"out": (h, U * h.abs() + eu * f.abs() + 1.2 * u.abs() * ez + 2.0 ** -18 * (u * z).abs() + 1e-30)}
    r["hg"] = (torch.cat([u, z], 1), torch.cat([U * u.abs() + eu, U * z.abs() + ez], 1) + 1e-30)
    du, dz = dh * f, dh * u * s
    su, sz = U * u.abs() + eu, U * z.abs() + ez
    tu = dh.abs() * (1.2 * sz + 2.0 ** -18 * z.abs())
    tz = dh.abs() * (1.2 * su + 1.2 * u.abs() * sz + 2.0 ** -18 * u.abs() * (1 + z.abs()))
    r["db_val"] = (du.sum(0), tu.sum(0) + FP * du.abs().sum(0) + U * du.sum(0).abs() + 1e-30)
    r["db_gate"] = (dz.sum(0), tz.sum(0) + FP * dz.abs().sum(0) + U * dz.sum(0).abs() + 1e-30)
    tu, tz = tu + (U + FP) * du.abs(), tz + (U + FP) * dz.abs()
    dx = du @ wv + dz @ wg
    r["dx"] = (dx, tu @ wv.abs() + tz @ wg.abs() + U * dx.abs() + 1e-30)
    xa = x.abs()
    for n, d, t in (("dw_val", du, tu), ("dw_gate", dz, tz)):
        w = d.t().contiguous() @ x
        r[n] = (w, t.t().contiguous() @ xa + U * w.abs() + 1e-30)
    return r


def _near(got, want, name):
    assert torch.isfinite(got).all(), name
    d = (got.double() - want[0]).abs()
    assert float(d.norm()) <= 6 * U * float(want[0].norm()) + 1e-20, f"{name}: relative error {float(d.norm() / want[0].norm()):.3g}"
    assert (d <= want[1]).all(), f"{name}: worst over its bound by {float((d - want[1]).max()):.3g}"


def _make(M, K, F, *, bias=False, fused=False, pitch=0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF16)

    def padded(r, c, **kw):  # a view whose rows are `pitch` further apart, NaN between them
        if not pitch:
            return rnd(r, c, **kw)
        b = torch.full((r, c + pitch), float("nan"), dtype=BF16, device="cuda")
        b[:, :c] = rnd(r, c, **kw)
        return b[:, :c]

    x, dh = padded(M, K), padded(M, F)
    if fused:  # [value | gate] of one matrix, as GEGLU's projection has them
        w = padded(2 * F, K, std=K ** -0.5)
        wv, wg = w[:F], w[F:]
    else:
        wv, wg = padded(F, K, std=K ** -0.5), padded(F, K, std=1.5 * K ** -0.5)
    bv, bg = (rnd(F, std=0.3), rnd(F, std=0.3)) if bias else (None, None)
    e = lambda r, c: torch.full((r, c + pitch), 7.0, dtype=BF16, device="cuda")[:, :c]  # noqa: E731
    res = dict(out=e(M, F), hg=e(M, 2 * F), dx=e(M, K), dw_val=e(F, K), dw_gate=e(F, K))
    if bias:
        res.update(db_val=torch.full((F,), 7.0, dtype=BF16, device="cuda"), db_gate=torch.full((F,), 7.0, dtype=BF16, device="cuda"))
    return x, wv, wg, bv, bg, dh, res


def _step(x, wv, wg, bv, bg, dh, res, act):
    from ai_toolkit_amd import ops

    ops.gated_ffn_fwd(x, wv, wg, res["out"], act=act, b_val=bv, b_gate=bg, hg=res["hg"])
    ops.gated_ffn_bwd(dh, x, wv, wg, res["hg"], act=act, **{k: v for k, v in res.items() if k.startswith("d")})


def _case(M, K, F, *, act="gelu_tanh", **kw):
    a = _make(M, K, F, **kw)
    want = _want(*a[:6], act)
    _step(*a, act)
    torch.cuda.synchronize()
    for n, t in a[6].items():
        _near(t, want[n], n)
        if t.dim() == 2 and t.stride(0) > t.shape[1]:  # the gaps between the rows stay as they were
            gap = torch.as_strided(t, (t.shape[0], t.stride(0) - t.shape[1]), (t.stride(0), 1), t.storage_offset() + t.shape[1])[:-1]
            assert (gap == 7.0).all(), n
    return a, want


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 33, 64, 100, 127, 129, 200, 300])
@pytest.mark.parametrize("K,F", [(64, 64), (8, 8), (72, 136), (200, 328), (512, 1024)])
def test_sizes(M, K, F):
    _case(M, K, F, seed=M)


# the last three: a last round of half tiles, some of them with a few rows or none
@pytest.mark.parametrize("M,K,F", [(2048, 512, 4096), (4096, 640, 2560), (600, 1000, 10240), (2300, 328, 4104), (2100, 136, 4104), (900, 72, 2560)])
@pytest.mark.parametrize("act", ["gelu_tanh", "gelu", "silu"])
def test_large_tiles(M, K, F, act):
    _case(M, K, F, act=act, bias=act == "gelu")


# more strips of the weights than a launch for few rows takes, fewer tiles than compute units
@pytest.mark.parametrize("M,K,F", [(600, 136, 1000), (130, 72, 4104), (700, 8, 1032), (129, 520, 6000), (1000, 768, 2048)])
@pytest.mark.parametrize("bias,fused,pitch", [(False, False, 0), (True, True, 40)])
def test_small_tiles(M, K, F, bias, fused, pitch):
    _case(M, K, F, bias=bias, fused=fused, pitch=pitch, act="gelu" if bias else "silu")


@pytest.mark.parametrize("act", ["gelu_tanh", "gelu", "silu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("pitch", [0, 40])
def test_forms(act, bias, fused, pitch):
    _case(150, 136, 264, act=act, bias=bias, fused=fused, pitch=pitch)


def test_without_saving_and_with_one_gradient_at_a_time():
    from ai_toolkit_amd import ops

    (x, wv, wg, bv, bg, dh, res), want = _case(170, 320, 640, bias=True, act="gelu")
    out = torch.zeros_like(res["out"])
    ops.gated_ffn_fwd(x, wv, wg, out, act="gelu", b_val=bv, b_gate=bg)
    assert torch.equal(out, res["out"])
    for n in ("dx", "dw_val", "dw_gate", "db_val", "db_gate"):
        one = torch.zeros_like(res[n])
        ops.gated_ffn_bwd(dh, x, wv, wg, res["hg"], act="gelu", **{n: one})
        assert torch.equal(one, res[n]), n
    ops.gated_ffn_bwd(dh, x, wv, wg, res["hg"], act="gelu")  # nothing asked for: nothing happens


def test_agrees_with_the_gemm_and_geglu_calls():
    """the same block through gemm_nt and geglu_fwd, which round the projections to bf16 in between: two roundings apart at most (u of value and gate, |act'| < 1.2)"""
    from ai_toolkit_amd import ops

    x, wv, wg, bv, bg, dh, res = _make(512, 640, 2560, fused=True)
    ops.gated_ffn_fwd(x, wv, wg, res["out"], act="gelu")
    hg = torch.empty(512, 5120, dtype=BF16, device="cuda")
    ops.gemm_nt(x, torch.cat([wv, wg]), hg)
    two = torch.empty(512, 2560, dtype=BF16, device="cuda")
    ops.geglu_fwd(hg, two)
    assert float((two.double() - res["out"].double()).norm() / two.double().norm()) <= 4 * U


def test_values_that_are_not_finite_stay_in_their_row():
    from ai_toolkit_amd import ops

    x, wv, wg, bv, bg, dh, res = _make(300, 200, 328)
    x[7, 3] = float("nan")
    ops.gated_ffn_fwd(x, wv, wg, res["out"])
    assert [i for i in range(300) if not bool(torch.isfinite(res["out"][i]).all())] == [7]


def test_large_gates_saturate():
    from ai_toolkit_amd import ops

    x, wv, wg, bv, bg, dh, res = _make(40, 64, 72)
    for act in ("gelu_tanh", "gelu", "silu"):
        for sign in (1.0, -1.0):
            big = torch.full((72,), sign * 1e4, dtype=BF16, device="cuda")
            one = torch.ones(72, dtype=BF16, device="cuda")
            ops.gated_ffn_fwd(torch.zeros_like(x), wv, wg, res["out"], act=act, b_val=one, b_gate=big, hg=res["hg"])
            assert bool((res["out"].float() == (big.float() if sign > 0 else 0.0)).all()), (act, sign)
            ops.gated_ffn_bwd(dh, x, wv, wg, res["hg"], act=act, dx=res["dx"], dw_val=res["dw_val"], dw_gate=res["dw_gate"])
            assert all(bool(torch.isfinite(res[n]).all()) for n in ("dx", "dw_val", "dw_gate"))


def test_no_rows():
    from ai_toolkit_amd import ops

    x, wv, wg, bv, bg, dh, res = _make(3, 64, 72)
    ops.gated_ffn_fwd(x[:0], wv, wg, res["out"][:0], hg=res["hg"][:0])
    ops.gated_ffn_bwd(dh[:0], x[:0], wv, wg, res["hg"][:0], dx=res["dx"][:0], dw_val=res["dw_val"])
    assert bool((res["dw_val"] == 0).all())


def test_gradients_against_differences():
    x, wv, wg, bv, bg, dh, res = _make(50, 72, 64, bias=True)
    _step(x, wv, wg, bv, bg, dh, res, "gelu_tanh")
    want = _want(x, wv, wg, bv, bg, dh, "gelu_tanh")
    g = torch.Generator(device="cuda").manual_seed(5)
    base = [t.double() for t in (x, wv, wg, bv, bg)]
    for i, n in enumerate(("dx", "dw_val", "dw_gate", "db_val", "db_gate")):
        d = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)

        def loss(h):
            y = [t + h * d if j == i else t for j, t in enumerate(base)]
            return float(((y[0] @ y[1].t() + y[3]) * _act(y[0] @ y[2].t() + y[4], "gelu_tanh")[0] * dh.double()).sum())

        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        assert abs(float((res[n].double() * d).sum()) - slope) <= float((want[n][1] * d.abs()).sum()) + 1e-6 * abs(slope), n


@pytest.mark.parametrize("M,K,F", [(3, 512, 1024), (140, 200, 328), (2048, 512, 4096)])
def test_repeats_bit_for_bit_on_another_stream_and_in_replayed_graphs(M, K, F):
    sets = [_make(M, K, F, bias=True, seed=s) for s in (1, 2)]
    for a in sets:
        _step(*a, "gelu")
    torch.cuda.synchronize()
    want = [{n: t.clone() for n, t in a[6].items()} for a in sets]
    side = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(side):
        for a, w in zip(sets, want):
            for t in a[6].values():
                t.zero_()
            _step(*a, "gelu")
        side.synchronize()
        assert all(torch.equal(t, w[n]) for a, w in zip(sets, want) for n, t in a[6].items())
        for a in sets:
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                _step(*a, "gelu")
            graphs.append(gr)
    torch.cuda.synchronize()
    for rep in range(4):
        for a in sets:
            for t in a[6].values():
                t.fill_(rep)
        for gr in graphs if rep % 2 else graphs[::-1]:
            gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, w[n]) for a, w in zip(sets, want) for n, t in a[6].items()), rep
        _step(*sets[0], "gelu")
