"""Cases for timing and checking three operators of this package around a transformer block:

  linear         linear_act: out = residual + act(x W^T + bias), forward alone or with every gradient
  qk_norm_rope   per-head rms norm of queries and keys and the position rotation, forward alone or with the gradients
  distill        distill_topk / distill_topk_fwd_bwd: the loss against a teacher's top logits, with or without its gradient

`run` computes a case either through the package (`own`) or in a plain form of elementary torch operations in 32 bits;
`exact` computes it from the definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
ACTS = ("none", "relu2", "gelu", "gelu_tanh", "silu")
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1.1920928955078125e-07          # the package's rms norms add the machine epsilon of fp32


# ---------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one token of a generation loop through an up projection of the 1024 / 4096 model
        dict(name="linear_token", op="linear", M=1, K=1024, N=4096, act="gelu", bias=True, residual=False, grad=False),
        # a dozen sequences generated together, the down projection that adds to the residual stream
        dict(name="linear_few", op="linear", M=12, K=4096, N=1024, act="none", bias=True, residual=True, grad=False),
        # an odd number of prompt tokens through layers whose widths divide nothing
        dict(name="linear_odd", op="linear", M=1531, K=1004, N=2311, act="silu", bias=True, residual=True, grad=False),
        # the 65536-token batch of the 1024 / 4096 model through its up projection
        dict(name="linear_batch", op="linear", M=65536, K=1024, N=4096, act="relu2", bias=True, residual=False, grad=False),
        # training step of the attention output projection at the 49152-token batch of the 768 model
        dict(name="linear_train_out", op="linear", M=49152, K=768, N=768, act="none", bias=True, residual=True, grad=True),
        # training step of an up projection with a smooth activation
        dict(name="linear_train_up", op="linear", M=16384, K=1024, N=4096, act="gelu_tanh", bias=True, residual=False, grad=True),
        # 16 sequences, one new token each, far positions
        dict(name="rope_token", op="rope", B=16, T=1, Hq=16, Hk=4, D=128, R=128, P=131072, dtype="bf16", packed=True,
             weights=True, interleaved=False, positions=True, grad=False),
        # training step at the 49152-token batch: 6 heads of 128, half of each head rotated, taken out of the packed projection
        dict(name="rope_train", op="rope", B=1, T=49152, Hq=6, Hk=6, D=128, R=64, P=65536, dtype="bf16", packed=True,
             weights=False, interleaved=False, positions=False, grad=True),
        # shared key heads, learned gains, pairs rotated, packed documents (positions given), 32-bit activations
        dict(name="rope_train_odd", op="rope", B=3, T=2731, Hq=12, Hk=4, D=80, R=80, P=4099, dtype="f32", packed=False,
             weights=True, interleaved=True, positions=True, grad=True),
        # loss of a handful of rows, no gradient
        dict(name="distill_few", op="distill", T=7, V=50304, K=20, dtype="bf16", ids64=True, cap=True, tail=False, weighted=False,
             temperature=1.0, mode="loss"),
        # training step: softcapped logits of the 50304-entry vocabulary, 64 entries of the teacher a row, loss and gradient at once
        dict(name="distill_train", op="distill", T=8192, V=50304, K=64, dtype="bf16", ids64=False, cap=True, tail=False,
             weighted=False, temperature=1.0, mode="fused"),
        # 32-bit logits with masked padding columns, the teacher's remaining mass kept, padded rows, through autograd
        dict(name="distill_tail", op="distill", T=1003, V=50257, K=100, dtype="f32", ids64=True, cap=False, tail=True, weighted=True,
             temperature=2.0, mode="autograd"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size spread over the logarithm of lo .. hi: as drawn, or rounded to a multiple of 8 or of 64."""
    n = _log_int(rng, lo, hi)
    step = rng.choice((1, 8, 64))
    return min(hi, max(lo, n // step * step)) if n >= step else n


def draw(rng):
    op = rng.choice(("linear", "rope", "distill"))
    if op == "linear":
        grad = rng.random() < 0.5
        K, N = _size(rng, 64, 4096), _size(rng, 64, 4096)
        most = 65536 * 1024 * 4096 // (6 if grad else 2)
        M = _log_int(rng, 1, max(1, min(65536, most // (K * N))))
        return dict(op=op, M=M, K=K, N=N, act=rng.choice(ACTS), bias=rng.random() < 0.7, residual=rng.random() < 0.5, grad=grad)
    if op == "rope":
        D = rng.choice((64, 128, 128, rng.randrange(16, 257, 2), rng.randrange(16, 257, 8)))
        Hk = rng.choice((1, 2, 4, 6, 8))
        Hq = Hk * rng.choice((1, 1, 2, 3, 4))
        B = _log_int(rng, 1, 16)
        dtype = rng.choice(("bf16", "bf16", "f32"))
        most = 49152 * 12 * 128 // ((Hq + Hk) * D * (2 if dtype == "f32" else 1))
        T = _log_int(rng, 1, max(1, min(49152, most) // B))
        positions = rng.random() < 0.5
        R = D if rng.random() < 0.6 else rng.randrange(2, D + 1, 2)
        return dict(op=op, B=B, T=T, Hq=Hq, Hk=Hk, D=D, R=R, P=max(T, _log_int(rng, 2048, 131072)), dtype=dtype,
                    packed=rng.random() < 0.5, weights=rng.random() < 0.5, interleaved=rng.random() < 0.5, positions=positions,
                    grad=rng.random() < 0.7)
    V = rng.choice((50304, 50257, _size(rng, 1000, 131072)))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    T = _log_int(rng, 1, max(1, 8192 * 50304 // (V * (2 if dtype == "f32" else 1))))
    return dict(op=op, T=T, V=V, K=_log_int(rng, 1, 128), dtype=dtype, ids64=rng.random() < 0.5, cap=rng.random() < 0.5,
                tail=rng.random() < 0.5, weighted=rng.random() < 0.5, temperature=rng.choice((1.0, 1.0, 2.0, 0.7)),
                mode=rng.choice(("loss", "fused", "autograd")))


def work(case):
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        rows_n = 1 + int(case["residual"])
        nbytes = 2 * (M * K + N * K + rows_n * M * N + int(case["bias"]) * N)
        flops = 2 * M * K * N
        if case["grad"]:           # dout in; dx, dW, dbias out (the residual's gradient is dout itself)
            nbytes += 2 * (M * N + M * K + N * K + int(case["bias"]) * N)
            flops *= 3
        return dict(bytes=nbytes, flops=flops)
    if case["op"] == "rope":
        tokens, size = case["B"] * case["T"], DTYPES[case["dtype"]].itemsize
        n = tokens * (case["Hq"] + case["Hk"]) * case["D"]
        nbytes = 2 * n * size + min(tokens, case["P"]) * case["R"] * 4 + tokens * 8 * int(case["positions"])
        if case["grad"]:           # x is still wanted: dout in, dx out
            nbytes += 2 * n * size
        return dict(bytes=nbytes, flops=(24 if case["grad"] else 8) * n)
    T, V, K = case["T"], case["V"], case["K"]
    size = DTYPES[case["dtype"]].itemsize
    ids = 8 if case["ids64"] else 4
    nbytes = T * V * size + T * K * (4 + ids) + 4 * T * (1 + int(case["tail"]) + int(case["weighted"]))
    flops = T * V * (10 if case["cap"] else 4)
    if case["mode"] != "loss":
        nbytes += T * V * size
        flops *= 2
    return dict(bytes=nbytes, flops=flops)


# ---------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return dict(case=dict(case), **{"linear": _prep_linear, "rope": _prep_rope, "distill": _prep_distill}[case["op"]](case, g))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _prep_linear(c, g):
    bf = torch.bfloat16
    M, K, N, grad = c["M"], c["K"], c["N"], c["grad"]
    s = dict(x=_randn(g, M, K, dtype=bf), w=_randn(g, N, K, dtype=bf, scale=K ** -0.5),
             bias=_randn(g, N, dtype=bf, scale=0.5) if c["bias"] else None,
             residual=_randn(g, M, N, dtype=bf) if c["residual"] else None,
             dout=_randn(g, M, N, dtype=bf) if grad else None)
    if grad:
        for k in ("x", "w", "bias", "residual"):
            if s[k] is not None:
                s[k].requires_grad_()
    return s


def _prep_rope(c, g):
    dt = DTYPES[c["dtype"]]
    B, T, Hq, Hk, D, R, P = (c[k] for k in ("B", "T", "Hq", "Hk", "D", "R", "P"))
    if c["packed"]:                 # queries, keys and values side by side, as one projection leaves them
        qkv = _randn(g, B, T, Hq + 2 * Hk, D, dtype=dt)
        q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
    else:
        q, k = _randn(g, B, T, Hq, D, dtype=dt), _randn(g, B, T, Hk, D, dtype=dt)
    freq = (1.0 / 10000.0) ** (torch.arange(R // 2, device=DEV, dtype=torch.float64) * 2 / R)
    angle = torch.arange(P, device=DEV, dtype=torch.float64)[:, None] * freq
    positions = None
    if c["positions"]:              # documents of their own offsets
        start = torch.randint(0, P - T + 1, (B, 1), generator=g, device=DEV)
        positions = start + torch.arange(T, device=DEV)
    s = dict(q=q, k=k, cos=angle.cos().float(), sin=angle.sin().float(), positions=positions,
             q_weight=(1 + _randn(g, D, scale=0.2)).to(dt) if c["weights"] else None,
             k_weight=(1 + _randn(g, D, scale=0.2)).to(dt) if c["weights"] else None,
             dq=_randn(g, B, T, Hq, D, dtype=dt) if c["grad"] else None,
             dk=_randn(g, B, T, Hk, D, dtype=dt) if c["grad"] else None)
    if c["grad"]:
        s["q"], s["k"] = s["q"].detach(), s["k"].detach()
        for name in ("q", "k", "q_weight", "k_weight"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def _prep_distill(c, g):
    dt = DTYPES[c["dtype"]]
    T, V, K = c["T"], c["V"], c["K"]
    logits = torch.randn(T, V, generator=g, device=DEV)
    logits.mul_(2.5)
    # distinct ids: a start and a step for every row; the teacher likes what the student likes, roughly
    step = torch.randint(1, max(2, V // K), (T, 1), generator=g, device=DEV)
    ids = (torch.randint(0, V, (T, 1), generator=g, device=DEV) + step * torch.arange(K, device=DEV)) % V
    teacher = (_randn(g, T, K, scale=1.5) + 9.0 - 3.0 * torch.arange(1, K + 1, device=DEV).float().log()).sort(1, descending=True)[0]
    logits.scatter_add_(1, ids, teacher * 0.8 + _randn(g, T, K))
    if not c["cap"] and V > 1000:   # padding columns masked out
        first = V - V % 64 if V % 64 else V - 47
        masked = torch.arange(V, device=DEV) >= first
        keep = torch.zeros(T, V, dtype=torch.bool, device=DEV).scatter_(1, ids, True)
        logits.masked_fill_(masked & ~keep, float("-inf"))
    logits = logits.to(dt)
    lse = None
    if c["tail"]:                   # 3 to 30 % of the teacher's mass lies outside its list
        rest = 0.03 + 0.27 * torch.rand(T, generator=g, device=DEV)
        lse = torch.logsumexp(teacher / c["temperature"], 1) - torch.log1p(-rest)
    weight = None
    if c["weighted"]:               # an eighth of the rows are padding
        weight = torch.rand(T, generator=g, device=DEV) + 0.5
        weight = torch.where(torch.rand(T, generator=g, device=DEV) < 0.125, torch.zeros_like(weight), weight)
    s = dict(logits=logits, ids=ids if c["ids64"] else ids.int(), teacher=teacher, lse=lse, weight=weight)
    if c["mode"] == "autograd":
        s["logits"].requires_grad_()
        s["dloss"] = torch.rand(T, generator=g, device=DEV) / T
    return s


CAP = (23.0, 5.0, 7.5)              # the model's softcap: 23 sigmoid((l + 5) / 7.5)


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    return {"linear": _run_linear, "rope": _run_rope, "distill": _run_distill}[state["case"]["op"]](state)


def _act(z, act):
    """(act(z), act'(z)) written out."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu2":
        r = z.clamp_min(0)
        return r * r, 2 * r
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * 0.7071067811865476))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    if act == "gelu_tanh":
        u = 0.7978845608028654 * (z + 0.044715 * z * z * z)
        t = torch.tanh(u)
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * 0.7978845608028654 * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return z * s, s * (1 + z * (1 - s))


def _run_linear(s):
    c = s["case"]
    x, w, bias, residual = s["x"], s["w"], s["bias"], s["residual"]
    if own:
        import modded_nanogpt_amd as amd
        out = amd.linear_act(x, w, bias, residual, c["act"])
        if not c["grad"]:
            return {"out": out}
        names = [n for n in ("x", "w", "bias", "residual") if s[n] is not None]
        grads = torch.autograd.grad(out, [s[n] for n in names], s["dout"])
        return {"out": out.detach(), **{"d" + n: v for n, v in zip(names, grads)}}
    with torch.no_grad():
        bf = torch.bfloat16
        xf, wf = x.float(), w.float()
        z = xf @ wf.t()
        if bias is not None:
            z = z + bias.float()
        y, slope = _act(z, c["act"])
        out = (y if residual is None else y + residual.float()).to(bf)
        if not c["grad"]:
            return {"out": out}
        dz = s["dout"].float() * slope
        res = {"out": out, "dx": (dz @ wf).to(bf), "dw": (dz.t() @ xf).to(bf)}
        if bias is not None:
            res["dbias"] = dz.sum(0).to(bf)
        if residual is not None:
            res["dresidual"] = s["dout"]
        return res


def _rotate(x, cos, sin, R, interleaved, back=False):
    if back:
        sin = -sin
    rot, rest = x[..., :R], x[..., R:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = rot[..., :R // 2], rot[..., R // 2:]
        rot = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((rot, rest), -1)


def _run_rope(s):
    c = s["case"]
    if own:
        import modded_nanogpt_amd as amd
        q, k = amd.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], q_weight=s["q_weight"],
                                k_weight=s["k_weight"], eps=EPS, interleaved=c["interleaved"])
        if not c["grad"]:
            return {"q": q, "k": k}
        names = [n for n in ("q", "k", "q_weight", "k_weight") if s[n] is not None]
        grads = torch.autograd.grad((q, k), [s[n] for n in names], (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), **{"d" + n: v for n, v in zip(names, grads)}}
    with torch.no_grad():
        R, D = c["R"], c["D"]
        if s["positions"] is None:
            cos, sin = s["cos"][:c["T"]], s["sin"][:c["T"]]
        else:
            cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
        res = {}
        for n in ("q", "k"):
            x, w = s[n].float(), s[n + "_weight"]
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            xn = x * r
            y = xn if w is None else xn * w.float()
            res[n] = _rotate(y, cos, sin, R, c["interleaved"]).to(s[n].dtype)
            if c["grad"]:
                g = _rotate(s["d" + n].float(), cos, sin, R, c["interleaved"], back=True)
                if w is not None:
                    res["d" + n + "_weight"] = (g * xn).sum((0, 1, 2)).to(w.dtype)
                    g = g * w.float()
                res["d" + n] = (r * (g - xn * (g * xn).mean(-1, keepdim=True))).to(s[n].dtype)
        order = ["q", "k"] + (["dq", "dk"] + (["dq_weight", "dk_weight"] if c["weights"] else []) if c["grad"] else [])
        return {n: res[n] for n in order}


def _run_distill(s):
    c = s["case"]
    cap = CAP if c["cap"] else None
    tau = c["temperature"]
    if own:
        import modded_nanogpt_amd as amd
        kw = dict(teacher_lse=s["lse"], row_weight=s["weight"], temperature=tau, softcap=cap)
        if c["mode"] == "fused":
            losses, grad = amd.distill_topk_fwd_bwd(s["logits"], s["ids"], s["teacher"], grad_scale=1.0 / c["T"], **kw)
            return {"losses": losses, "dlogits": grad}
        losses = amd.distill_topk(s["logits"], s["ids"], s["teacher"], **kw)
        if c["mode"] == "loss":
            return {"losses": losses}
        (grad,) = torch.autograd.grad(losses, [s["logits"]], s["dloss"])
        return {"losses": losses.detach(), "dlogits": grad}
    with torch.no_grad():
        l = s["logits"].float()
        ids = s["ids"].long()
        if cap is not None:
            sg = 1 / (1 + torch.exp(-(l + cap[1]) / cap[2]))
            z = cap[0] * sg / tau
        else:
            z = l / tau
        top = z.max(1, keepdim=True)[0]
        e = torch.exp(z - top)
        total = e.sum(1, keepdim=True)
        logq = z.gather(1, ids) - top - total.log()
        t = s["teacher"].double() / tau          # the mass outside the list is a small difference of numbers near 1
        if s["lse"] is None:
            t = t - t.max(1, keepdim=True)[0]
            logp = t - t.exp().sum(1, keepdim=True).log()
        else:
            logp = t - s["lse"].double()[:, None]
        p = logp.exp()
        kl = (p * (logp - logq.double())).sum(1)
        if s["lse"] is not None:
            rest_p = (1 - p.sum(1)).clamp_min(0)
            rest_e = e.scatter(1, ids, 0.0).sum(1)
            logq_rest = rest_e.log() - total[:, 0].log()
            kl = kl + rest_p * (rest_p.log() - logq_rest.double())
        w = torch.ones_like(total[:, 0]) if s["weight"] is None else s["weight"]
        losses = (tau * tau * w * kl).float()
        if c["mode"] == "loss":
            return {"losses": losses}
        rows = (w / c["T"] if c["mode"] == "fused" else w * s["dloss"]) * tau
        if s["lse"] is None:
            grad = e / total
        else:
            grad = e * ((1 - rest_p.float() * total[:, 0] / rest_e) / total[:, 0])[:, None]
            grad.scatter_(1, ids, e.gather(1, ids) / total)
        grad.scatter_add_(1, ids, -p.float())
        grad = grad * rows[:, None]
        if cap is not None:
            grad = grad * (cap[0] / cap[2] * sg * (1 - sg))
        return {"losses": losses, "dlogits": grad.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "rope": _exact_rope, "distill": _exact_distill}[case["op"]](case, s)


def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_()


def _exact_linear(c, s):
    F = torch.nn.functional
    fn = {"none": lambda z: z, "relu2": lambda z: F.relu(z).square(), "gelu": F.gelu,
          "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}[c["act"]]
    ins = {n: _leaf(s[n]) for n in ("x", "w", "bias", "residual") if s[n] is not None}
    with torch.set_grad_enabled(c["grad"]):
        out = fn(F.linear(ins["x"], ins["w"], ins.get("bias")))
        if "residual" in ins:
            out = out + ins["residual"]
    if not c["grad"]:
        return {"out": out}
    grads = torch.autograd.grad(out, list(ins.values()), s["dout"].double())
    return {"out": out.detach(), **{"d" + n: v for n, v in zip(ins, grads)}}


def _exact_rope(c, s):
    names = [n for n in ("q", "k", "q_weight", "k_weight") if s[n] is not None]
    ins = {n: _leaf(s[n]) for n in names}
    half = c["R"] // 2
    pos = torch.arange(c["T"], device=DEV).expand(c["B"], -1) if s["positions"] is None else s["positions"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, :, None]
    outs = []
    with torch.set_grad_enabled(c["grad"]):
        for n in ("q", "k"):
            x = ins[n]
            y = x / (x.pow(2).sum(-1, keepdim=True) / c["D"] + EPS).sqrt()
            if n + "_weight" in ins:
                y = y * ins[n + "_weight"]
            if c["interleaved"]:
                pairs = torch.view_as_complex(y[..., :c["R"]].unflatten(-1, (half, 2)).contiguous()) * turn
                rot = torch.view_as_real(pairs).flatten(-2)
            else:
                pairs = torch.complex(y[..., :half], y[..., half:c["R"]]) * turn
                rot = torch.cat((pairs.real, pairs.imag), -1)
            outs.append(torch.cat((rot, y[..., c["R"]:]), -1))
    if not c["grad"]:
        return {"q": outs[0], "k": outs[1]}
    grads = torch.autograd.grad(outs, list(ins.values()), (s["dq"].double(), s["dk"].double()))
    return {"q": outs[0].detach(), "k": outs[1].detach(), **{"d" + n: v for n, v in zip(names, grads)}}


def _exact_distill(c, s):
    tau, V, T = c["temperature"], c["V"], c["T"]
    losses, grads = [], []
    rows = max(1, 2 ** 25 // V)
    for a in range(0, T, rows):
        sl = slice(a, min(T, a + rows))
        l = _leaf(s["logits"][sl])
        ids, t = s["ids"][sl].long(), s["teacher"][sl].double() / tau
        w = torch.ones(l.shape[0], device=DEV, dtype=torch.float64) if s["weight"] is None else s["weight"][sl].double()
        with torch.set_grad_enabled(c["mode"] != "loss"):
            z = l if not c["cap"] else CAP[0] * torch.sigmoid((l + CAP[1]) / CAP[2])
            logq = torch.log_softmax(z / tau, 1)
            if s["lse"] is None:
                logp = torch.log_softmax(t, 1)
                kl = (logp.exp() * (logp - logq.gather(1, ids))).sum(1)
            else:
                logp = t - s["lse"][sl].double()[:, None]
                rest_p = 1 - logp.exp().sum(1)
                others = logq.scatter(1, ids, float("-inf"))
                kl = (logp.exp() * (logp - logq.gather(1, ids))).sum(1)
                kl = kl + rest_p * (rest_p.log() - torch.logsumexp(others, 1))
            loss = tau * tau * w * kl
        losses.append(loss.detach())
        if c["mode"] != "loss":
            up = torch.full_like(loss, 1.0 / T) if c["mode"] == "fused" else s["dloss"][sl].double()
            grads.append(torch.autograd.grad(loss, l, up)[0])
    res = {"losses": torch.cat(losses)}
    if grads:
        res["dlogits"] = torch.cat(grads)
    return res
