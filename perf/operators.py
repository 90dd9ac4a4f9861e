"""What is measured of the text-encoder block's operators: attention with a learned relative position bias (forward, and forward with backward),
layer / RMS norm with the gradient of its weight, and the gated feed-forward projections with their gradients.

A case's "op" names the operator ("attn", "norm", "ffn"), "train" whether the pass is forward and backward or the forward alone."""
import math

import torch

own = False

BF16 = torch.bfloat16
DEV = "cuda"
D = 64  # head width of the text encoders (T5 / UMT5 d_kv, CLIP)


# ------------------------------------------------------------------------------------------------------------------ cases
def _attn(name, B, H, S, *, train=False, buckets=32, max_distance=128, bias=True, causal=False, len_lo=-1, len_hi=-1, scale=1.0):
    return {"name": name, "op": "attn", "train": train, "B": B, "H": H, "S": S, "buckets": buckets, "max_distance": max_distance, "bias": bias,
            "causal": causal, "len_lo": len_lo, "len_hi": len_hi, "scale": scale}


def _norm(name, M, C, *, train=False, rms=True, dres=False):
    return {"name": name, "op": "norm", "train": train, "M": M, "C": C, "rms": rms, "dres": dres}


def _ffn(name, M, K, F, *, train=False, act="gelu_tanh", bias=False):
    return {"name": name, "op": "ffn", "train": train, "M": M, "K": K, "F": F, "act": act, "bias": bias}


def listed():
    return [
        # a pair of CLIP prompts (positive and negative) through one layer: the latency of a short causal sequence, no position bias
        _attn("attn clip pair", 2, 12, 77, bias=False, causal=True, scale=0.125),
        # one FLUX prompt through a T5 layer: the trainer passes no mask, all 512 positions are attended
        _attn("attn t5 one prompt", 1, 64, 512),
        # a training batch of captions with their attention mask: lengths from a few words to the full window
        _attn("attn train captions", 4, 64, 512, train=True, len_lo=24, len_hi=512),
        # a small encoder on an odd window; one caption of the batch was dropped to nothing
        _attn("attn train odd", 3, 6, 333, train=True, len_lo=0, len_hi=333),
        # long captions, every position attended
        _attn("attn train long", 1, 32, 2048, train=True),
        # the final norm of a CLIP prompt
        _norm("norm clip", 77, 768, rms=False),
        # a T5 layer's norm over a training batch
        _norm("norm train t5", 4096, 4096, train=True, dres=True),
        # LayerNorm of a UNet transformer block or of a wide CLIP encoder over many rows, an odd number of them
        _norm("norm train many rows", 32761, 1280, train=True, rms=False),
        # four tokens through a small encoder's feed-forward block: the weights' way through the chip
        _ffn("ffn few tokens", 4, 512, 1024),
        # one FLUX prompt through a T5 feed-forward block
        _ffn("ffn t5 one prompt", 512, 4096, 10240),
        # a training batch of four prompts through it
        _ffn("ffn train t5", 2048, 4096, 10240, train=True),
        # an SDXL transformer block's feed-forward projection (erf GELU, biases) over 64 x 64 tokens
        _ffn("ffn train sdxl", 4096, 640, 2560, train=True, act="gelu", bias=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attn", "norm", "ffn"])
    train = rng.random() < 0.5
    if op == "attn":
        S = _log_int(rng, 1, 2048)
        H = rng.choice([1, 4, 6, 8, 12, 16, 20, 32, 64])
        B = max(1, min(rng.randint(1, 8), 32 * 2048 * 2048 // (H * S * S)))
        H = max(1, min(H, 32 * 2048 * 2048 // (B * S * S)))
        buckets, max_distance = rng.choice([(32, 128), (32, 128), (16, 64), (64, 256)])
        bias = rng.random() < 0.8
        masked = rng.random() < 0.6
        lo = rng.randint(0, S) if masked else -1
        return {k: v for k, v in _attn("", B, H, S, train=train, buckets=buckets, max_distance=max_distance, bias=bias, causal=rng.random() < 0.3,
                                       len_lo=lo, len_hi=rng.randint(lo, S) if masked else -1, scale=rng.choice([1.0, 0.125])).items() if k != "name"}
    if op == "norm":
        C = 8 * _log_int(rng, 8, 1024)
        M = _log_int(rng, 1, min(65536, 32761 * 1280 // C))
        rms = rng.random() < 0.5
        return {k: v for k, v in _norm("", M, C, train=train, rms=rms, dres=train and rng.random() < 0.5).items() if k != "name"}
    K = 8 * _log_int(rng, 8, 512)
    F = 8 * _log_int(rng, 8, 1280)
    M = _log_int(rng, 1, min(8192, 2048 * 4096 * 10240 // (K * F)))
    return {k: v for k, v in _ffn("", M, K, F, train=train, act=rng.choice(["gelu_tanh", "gelu", "silu"]), bias=rng.random() < 0.4).items() if k != "name"}


def _lens(case):
    """valid keys of each sample, a function of the case alone; None: no mask"""
    if case["len_lo"] < 0:
        return None
    B, lo, hi = case["B"], case["len_lo"], case["len_hi"]
    return [lo + (hi - lo) * b // max(1, B - 1) for b in range(B)]


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def rand(*shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    def empty(*shape, dtype=BF16):
        return torch.empty(*shape, dtype=dtype, device=DEV)

    s = {"case": case}
    if case["op"] == "attn":
        B, H, S = case["B"], case["H"], case["S"]
        std = 0.35 * case["scale"] ** -0.5  # logits of the size that an encoder's heads have
        # one projection's output: q, k and v are column blocks of it, as a program that fuses the three projections has them
        qkv = torch.cat([rand(B * S, H * D, std=std), rand(B * S, H * D, std=std), rand(B * S, H * D)], 1)
        s["q"], s["k"], s["v"] = qkv[:, :H * D], qkv[:, H * D:2 * H * D], qkv[:, 2 * H * D:]
        s["table"] = rand(case["buckets"], H, std=0.7) if case["bias"] else None
        lens = _lens(case)
        s["mask"] = None
        if lens is not None:
            s["mask"] = torch.arange(S, device=DEV)[None, :] < torch.tensor(lens, device=DEV)[:, None]
        s["o"], s["lse"] = empty(B * S, H * D), empty(B, H, S, dtype=torch.float32)
        if case["train"]:
            s["do"] = rand(B * S, H * D)
            dqkv = empty(B * S, 3 * H * D)
            s["dq"], s["dk"], s["dv"] = dqkv[:, :H * D], dqkv[:, H * D:2 * H * D], dqkv[:, 2 * H * D:]
            s["dtable"] = empty(case["buckets"], H) if case["bias"] else None
    elif case["op"] == "norm":
        M, C = case["M"], case["C"]
        # a residual stream: every column has its own scale and, for layer norm, its own mean
        x = torch.randn(M, C, generator=g, device=DEV) * (0.5 + torch.rand(C, generator=g, device=DEV))
        if not case["rms"]:
            x = x + 0.5 * torch.randn(C, generator=g, device=DEV)
        s["x"] = x.to(BF16)
        s["weight"] = (1.0 + 0.2 * torch.randn(C, generator=g, device=DEV)).to(BF16)
        s["bias"] = None if case["rms"] else rand(C, std=0.2)
        s["y"] = empty(M, C)
        if case["train"]:
            s["dy"] = rand(M, C)
            s["dres"] = rand(M, C) if case["dres"] else None
            s["mean"], s["rstd"] = (None if case["rms"] else empty(M, dtype=torch.float32)), empty(M, dtype=torch.float32)
            s["dx"], s["dweight"] = empty(M, C), empty(C, dtype=torch.float32)
            s["dbias"] = None if case["rms"] else empty(C, dtype=torch.float32)
    else:
        M, K, F = case["M"], case["K"], case["F"]
        s["x"] = rand(M, K)
        s["w_val"], s["w_gate"] = rand(F, K, std=K ** -0.5), rand(F, K, std=1.5 * K ** -0.5)
        s["b_val"], s["b_gate"] = (rand(F, std=0.1), rand(F, std=0.1)) if case["bias"] else (None, None)
        s["out"] = empty(M, F)
        if case["train"]:
            s["dh"] = rand(M, F)
            s["hg"] = empty(M, 2 * F)
            s["dx"], s["dw_val"], s["dw_gate"] = empty(M, K), empty(F, K), empty(F, K)
            s["db_val"], s["db_gate"] = (empty(F), empty(F)) if case["bias"] else (None, None)
    return s


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    return (_run_own if own else _run_plain)[case["op"]](s, case)


def _own_attn(s, c):
    from ai_toolkit_amd import ops

    kw = dict(B=c["B"], H=c["H"], S=c["S"], scale=c["scale"], key_mask=s["mask"], max_distance=c["max_distance"], causal=c["causal"])
    ops.attn_relpos_fwd(s["q"], s["k"], s["v"], s["table"], s["o"], s["lse"], **kw)
    if not c["train"]:
        return [s["o"]]
    ops.attn_relpos_bwd(s["q"], s["k"], s["v"], s["table"], s["o"], s["lse"], s["do"], s["dq"], s["dk"], s["dv"], s["dtable"], **kw)
    return [s["o"], s["dq"], s["dk"], s["dv"]] + ([s["dtable"]] if c["bias"] else [])


def _own_norm(s, c):
    from ai_toolkit_amd import ops

    if not c["train"]:
        ops.norm_fwd(s["x"], s["weight"], s["y"], bias=s["bias"], rms=c["rms"], eps=1e-6)
        return [s["y"]]
    ops.norm_fwd(s["x"], s["weight"], s["y"], bias=s["bias"], rms=c["rms"], mean=s["mean"], rstd=s["rstd"], eps=1e-6)
    ops.norm_bwd(s["dy"], s["x"], s["weight"], s["rstd"], s["dx"], mean=s["mean"], rms=c["rms"], dres=s["dres"], dweight=s["dweight"], dbias=s["dbias"])
    return [s["y"], s["dx"], s["dweight"]] + ([] if c["rms"] else [s["dbias"]])


def _own_ffn(s, c):
    from ai_toolkit_amd import ops

    if not c["train"]:
        ops.gated_ffn_fwd(s["x"], s["w_val"], s["w_gate"], s["out"], act=c["act"], b_val=s["b_val"], b_gate=s["b_gate"])
        return [s["out"]]
    ops.gated_ffn_fwd(s["x"], s["w_val"], s["w_gate"], s["out"], act=c["act"], b_val=s["b_val"], b_gate=s["b_gate"], hg=s["hg"])
    ops.gated_ffn_bwd(s["dh"], s["x"], s["w_val"], s["w_gate"], s["hg"], act=c["act"], dx=s["dx"], dw_val=s["dw_val"], dw_gate=s["dw_gate"],
                      db_val=s["db_val"], db_gate=s["db_gate"])
    return [s["out"], s["dx"], s["dw_val"], s["dw_gate"]] + ([s["db_val"], s["db_gate"]] if c["bias"] else [])


_run_own = {"attn": _own_attn, "norm": _own_norm, "ffn": _own_ffn}


def _bucket_of(rel, buckets, max_distance, causal):
    """The bucket of every relative position rel = key - query: exact up to half of a sign's buckets, then by the logarithm up to max_distance, then
    the last one.  Causal: only the past has buckets.  In 64 bits with the border itself (an exact power) on the far side."""
    half = buckets if causal else buckets // 2
    base = torch.zeros_like(rel) if causal else (rel > 0).long() * half
    n = (-rel).clamp(min=0) if causal else rel.abs()
    exact_n = half // 2
    steps = torch.log(n.clamp(min=1).double() / exact_n) / math.log(max_distance / exact_n) * (half - exact_n)
    far = (exact_n + torch.floor(steps + 1e-9).long()).clamp(max=half - 1)
    return base + torch.where(n < exact_n, n, far)


def _plain_attn(s, c):
    B, H, S = c["B"], c["H"], c["S"]
    heads = lambda t: t.float().view(B, S, H, D).transpose(1, 2).contiguous()  # noqa: E731
    q, k, v = heads(s["q"]), heads(s["k"]), heads(s["v"])
    pos = torch.arange(S, device=DEV)
    rel = pos[None, :] - pos[:, None]
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * c["scale"]
    if c["bias"]:
        bucket = _bucket_of(rel, c["buckets"], c["max_distance"], c["causal"])
        score += s["table"].float()[bucket].permute(2, 0, 1)
    if c["causal"]:
        score.masked_fill_(rel > 0, float("-inf"))
    if s["mask"] is not None:
        score.masked_fill_(~s["mask"][:, None, None, :], float("-inf"))
    top = score.amax(3, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)  # a row with no key left: all probabilities are 0
    p = torch.exp(score - top)
    del score
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    rows = lambda t: t.transpose(1, 2).reshape(B * S, H * D).to(BF16)  # noqa: E731
    o = torch.matmul(p, v)
    if not c["train"]:
        return [rows(o)]
    do = heads(s["do"])
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (do * o).sum(3, keepdim=True))
    del dp, p
    dq = torch.matmul(ds, k) * c["scale"]
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * c["scale"]
    out = [rows(o), rows(dq), rows(dk), rows(dv)]
    if c["bias"]:
        # each diagonal of the summed [query, key] scores is one relative position: with the rows reversed and S more columns, row
        # r starts r places further right, so that the diagonals become columns.  64 bits: one bucket takes up to millions of terms
        skewed = torch.nn.functional.pad(ds.sum(0).flip(1), (0, S)).view(H, -1)[:, :S * (2 * S - 1)].view(H, S, 2 * S - 1)
        by_rel = skewed.sum(1, dtype=torch.float64)  # column j: key - query = j - (S - 1)
        all_rel = torch.arange(1 - S, S, device=DEV)
        member = torch.nn.functional.one_hot(_bucket_of(all_rel, c["buckets"], c["max_distance"], c["causal"]), c["buckets"]).double()
        out.append(torch.matmul(member.t().contiguous(), by_rel.t().contiguous()).to(BF16))
    return out


def _plain_norm(s, c):
    x, w = s["x"].float(), s["weight"].float()
    mean = 0.0 if c["rms"] else x.mean(1, keepdim=True)
    rstd = torch.rsqrt(((x - mean) ** 2).mean(1, keepdim=True) + 1e-6)
    xh = (x - mean) * rstd
    y = xh * w
    if not c["rms"]:
        y = y + s["bias"].float()
    if not c["train"]:
        return [y.to(BF16)]
    dy = s["dy"].float()
    g = dy * w
    dx = g - xh * (g * xh).mean(1, keepdim=True)
    if not c["rms"]:
        dx = dx - g.mean(1, keepdim=True)
    dx = dx * rstd
    if c["dres"]:
        dx = dx + s["dres"].float()
    out = [y.to(BF16), dx.to(BF16), (dy * xh).sum(0)]
    return out if c["rms"] else out + [dy.sum(0)]


def _act_and_slope(u, act):
    if act == "silu":
        z = torch.sigmoid(u)
        return u * z, z * (1 + u * (1 - z))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(u * math.sqrt(0.5)))
        return u * cdf, cdf + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    k0, k1 = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(k0 * (u + k1 * u ** 3))
    return 0.5 * u * (1 + t), 0.5 * (1 + t) + 0.5 * u * (1 - t * t) * k0 * (1 + 3 * k1 * u * u)


def _plain_ffn(s, c):
    x, wv, wg = s["x"].float(), s["w_val"].float(), s["w_gate"].float()
    uv, ug = torch.matmul(x, wv.t()), torch.matmul(x, wg.t())
    if c["bias"]:
        uv, ug = uv + s["b_val"].float(), ug + s["b_gate"].float()
    a, slope = _act_and_slope(ug, c["act"])
    out = (uv * a).to(BF16)
    if not c["train"]:
        return [out]
    dh = s["dh"].float()
    dv, dg = dh * a, dh * uv * slope
    dx = torch.matmul(dv, wv) + torch.matmul(dg, wg)
    outs = [out, dx.to(BF16), torch.matmul(dv.t(), x).to(BF16), torch.matmul(dg.t(), x).to(BF16)]
    return outs + [dv.sum(0).to(BF16), dg.sum(0).to(BF16)] if c["bias"] else outs


_run_plain = {"attn": _plain_attn, "norm": _plain_norm, "ffn": _plain_ffn}


# ------------------------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "attn":
        B, H, S = case["B"], case["H"], case["S"]
        lens = _lens(case) or [S] * B
        # query-key pairs that the masks leave
        pairs = sum(S * n - n * (n - 1) // 2 if case["causal"] else S * n for n in lens) * H
        rows, keys = B * S * H * D * 2, sum(lens) * H * D * 2
        table = case["buckets"] * H * 2 if case["bias"] else 0
        if not case["train"]:
            return {"bytes": 2 * rows + 2 * keys + table, "flops": 2 * 2 * D * pairs}
        # forward two products; backward five (the scores once more, dP, dV, dQ, dK): q, o, dO, dQ and k, v, dK, dV
        return {"bytes": 4 * rows + 2 * keys + 2 * rows + 2 * table, "flops": (2 + 5) * 2 * D * pairs}
    if case["op"] == "norm":
        M, C = case["M"], case["C"]
        if not case["train"]:
            return {"bytes": 2 * M * C * 2 + 2 * C, "flops": 6 * M * C}
        return {"bytes": (4 + (1 if case["dres"] else 0)) * M * C * 2 + 6 * C, "flops": 20 * M * C}
    M, K, F = case["M"], case["K"], case["F"]
    once = 2 * M * K * 2 * F
    if not case["train"]:
        return {"bytes": 2 * (M * K + 2 * F * K + M * F), "flops": once}
    # read x, both weights, dh; write h, dx and both weights' gradients
    return {"bytes": 2 * (2 * M * K + 2 * 2 * F * K + 2 * M * F), "flops": 3 * once}


# ------------------------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attn(s, case)
    leaf = lambda t: None if t is None else t.double().requires_grad_(case["train"])  # noqa: E731
    if case["op"] == "norm":
        x, w, b = leaf(s["x"]), leaf(s["weight"]), leaf(s["bias"])
        if case["rms"]:
            y = x / torch.sqrt(torch.mean(x * x, dim=1, keepdim=True) + 1e-6) * w
        else:
            y = torch.nn.functional.layer_norm(x, (case["C"],), w, b, 1e-6)
        if not case["train"]:
            return [y]
        found = torch.autograd.grad(y, [x, w] + ([] if b is None else [b]), s["dy"].double())
        dx = found[0] if s["dres"] is None else found[0] + s["dres"].double()
        return [y.detach(), dx] + list(found[1:])
    x, wv, wg, bv, bg = (leaf(s[n]) for n in ("x", "w_val", "w_gate", "b_val", "b_gate"))
    u, z = torch.nn.functional.linear(x, wv, bv), torch.nn.functional.linear(x, wg, bg)
    F = torch.nn.functional
    h = u * {"gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "gelu": F.gelu, "silu": F.silu}[case["act"]](z)
    if not case["train"]:
        return [h]
    leaves = [x, wv, wg] + ([bv, bg] if case["bias"] else [])
    return [h.detach()] + list(torch.autograd.grad(h, leaves, s["dh"].double()))


def _exact_buckets(case):
    """bucket of every distance 0 .. S - 1 of one sign, in whole numbers: distance n >= e is in step j >= 0 of the L logarithmic ones where
    (n / e) ** L >= (max_distance / e) ** j"""
    half = case["buckets"] if case["causal"] else case["buckets"] // 2
    e = half // 2
    L = half - e

    def of(n):
        if n < e:
            return n
        j = 0
        while j < L - 1 and n ** L * e ** (j + 1) >= case["max_distance"] ** (j + 1) * e ** L:
            j += 1
        return e + j

    return [of(n) for n in range(case["S"])], half


def _exact_attn(s, case):
    B, H, S = case["B"], case["H"], case["S"]
    train = case["train"]
    split = lambda t: t.double().view(B, S, H, D)  # noqa: E731
    q, k, v = split(s["q"]), split(s["k"]), split(s["v"])
    table = s["table"].double() if case["bias"] else None
    lens = _lens(case) or [S] * B
    index = None
    if case["bias"]:
        near, half = _exact_buckets(case)
        past = torch.tensor(near, device=DEV)
        # by key - query + S - 1; what lies ahead is the second half of the table, or masked
        ahead = torch.zeros_like(past) if case["causal"] else past + half
        line = torch.cat([past.flip(0), ahead[1:]])
        at = torch.arange(S, device=DEV)
        index = line[at[None, :] - at[:, None] + S - 1]
    o = torch.zeros(B, S, H, D, dtype=torch.float64, device=DEV)
    dq, dk, dv = (torch.zeros_like(o) for _ in range(3))
    dtable = None if table is None else torch.zeros_like(table)
    for b in range(B):
        n = lens[b]
        if n == 0:
            continue
        for h in range(H):
            qh, kh, vh = (t[b, :r, h].detach().clone().requires_grad_(train) for t, r in ((q, S), (k, n), (v, n)))
            a = qh @ kh.t() * case["scale"]
            th = None
            if table is not None:
                th = table[:, h].detach().clone().requires_grad_(train)
                a = a + th[index[:, :n]]
            if case["causal"]:
                a = a + torch.full((S, n), float("-inf"), dtype=torch.float64, device=DEV).triu(1)
            y = torch.softmax(a, 1) @ vh
            o[b, :, h] = y.detach()
            if train:
                found = torch.autograd.grad(y, [qh, kh, vh] + ([] if th is None else [th]), split(s["do"])[b, :, h])
                dq[b, :, h], dk[b, :n, h], dv[b, :n, h] = found[:3]
                if th is not None:
                    dtable[:, h] += found[3]
    rows = [t.reshape(B * S, H * D) for t in ((o, dq, dk, dv) if train else (o,))]
    return rows + ([dtable] if train and table is not None else [])
