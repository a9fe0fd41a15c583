"""Training next to `sageattn`: the operators' calls, their inputs, work and results.

Two operators, as one block of a transformer uses them around the framework's attention:

* `grad`: attention's backward pass, from the gradient of its output (and, where the caller merges
  parts by their logsumexp, of that) to those of Q, K and V; the probabilities are recomputed from
  the kept logsumexp;
* `norm`, `quant`, `norm_grad`: the root-mean-square norm with the residual's addition ahead of it,
  in 16 bits or as 8-bit codes with a scale per row for an 8-bit projection, and its gradients.

`listed()` names the calls that stand for real use, `draw(rng)` gives others of the same ranges.
`run` computes the plain form in 32 bits, or, where `own` is true, calls the framework.
"""
import os
import sys

import torch

#: whether `run` calls the framework's operators
own = False

EPS = 1e-6           # added to a row's mean square
FLOOR = 1e-12        # the least row scale

if not any(p.endswith("sageattention-rdna4_amd") for p in sys.path):
    sys.path.insert(0, os.path.join(os.getcwd(), "sageattention-rdna4_amd"))


# --------------------------------------------------------------------------------------- cases
def _grad(B, H, H_kv, N, N_kv, D, dtype, causal, layout="HND", dlse=False):
    return {"op": "grad", "B": B, "H": H, "H_kv": H_kv, "N": N, "N_kv": N_kv, "D": D,
            "dtype": dtype, "causal": causal, "layout": layout, "dlse": dlse}


def _norm(op, B, N, n, dtype, residual, H=0, codes=None, weight="same"):
    """B sequences of N rows of n values; with H, rows are heads of the first third of a fused
    projection. `residual`: one is added ahead (`norm_grad`: its gradient comes in as well)."""
    return {"op": op, "B": B, "N": N, "n": n, "dtype": dtype, "residual": residual, "H": H,
            "codes": codes, "weight": weight}


def listed():
    named = {
        # a short text, one sequence: launches and latency are most of it
        "grad_short": _grad(1, 8, 8, 257, 257, 64, "bf16", True),
        # image tokens on a caption's, for fine-tuning an image model: many queries, few keys
        "grad_cross": _grad(2, 10, 10, 4096, 77, 64, "fp16", False, layout="NHD"),
        # a 1024 x 1024 image's self-attention at head_dim 64
        "grad_image": _grad(2, 10, 10, 4096, 4096, 64, "fp16", False),
        # ragged length, with the gradient of the logsumexp, as attention over parts merges by it
        "grad_parts": _grad(1, 24, 24, 1777, 1777, 128, "fp16", True, dlse=True),
        # a batch of a language model's training step, grouped heads
        "grad_batch": _grad(4, 32, 8, 2048, 2048, 128, "bf16", True, layout="NHD"),
        # the same on one long document
        "grad_long": _grad(1, 32, 8, 16384, 16384, 128, "bf16", True),
        # one decoding step of a batch, residual added ahead of the norm: latency
        "norm_step": _norm("norm", 64, 1, 4096, "bf16", True),
        # the queries' heads normed, straight from a fused projection
        "norm_heads": _norm("norm", 2, 4001, 128, "bf16", False, H=32),
        # one decoding step into an int8 projection
        "quant_step": _norm("quant", 16, 1, 6144, "fp16", True, codes="int8"),
        # prompts into an e4m3 projection
        "quant_prompt": _norm("quant", 4, 4001, 4096, "bf16", True, codes="e4m3"),
        # the training step's gradients: of rows, residual and weight
        "norm_grad": _norm("norm_grad", 4, 4096, 4096, "bf16", True, weight="fp32"),
        # the same for heads of an image model's fused projection
        "norm_grad_heads": _norm("norm_grad", 2, 4250, 128, "fp16", False, H=24),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("grad", "grad", "grad", "norm", "quant", "norm_grad"))
    dtype = rng.choice(("fp16", "bf16"))
    if op == "grad":
        D = rng.choice((128, 128, 64))
        H_kv = rng.choice((1, 2, 8, 10))
        H = H_kv * rng.choice((1, 1, 4, 6))
        B = _size(rng, 1, 8)
        # at most an eighth of the queries times keys of the longest listed case
        most = min(16384, int((32 * 16384 * 16384 / 8 / (B * H)) ** 0.5))
        # 16 keys at least: a query that sees one key alone has gradients of zero, to be compared
        # with nothing but their own rounding
        causal = rng.random() < 0.5
        N_kv = _size(rng, 16, max(16, most))
        N = N_kv if causal or rng.random() < 0.4 else _size(rng, 1, most)
        return _grad(B, H, H_kv, N, N_kv, D, dtype, causal, rng.choice(("HND", "NHD")),
                     rng.random() < 0.3)
    weight = rng.choice(("same", "same", "fp32"))
    residual = rng.random() < 0.6
    codes = None
    if op == "quant":
        codes = "int8" if dtype == "fp16" and rng.random() < 0.7 else "e4m3"
    if rng.random() < 0.3:
        B, H, n = _size(rng, 1, 8), rng.choice((2, 8, 10, 24, 32)), rng.choice((64, 128))
        return _norm(op, B, _size(rng, 1, max(1, 1100000 // (B * H) * 64 // n)), n, dtype,
                     False, H, codes, weight)
    B, n = _size(rng, 1, 64), 8 * _size(rng, 2, 2048)
    return _norm(op, B, _size(rng, 1, max(1, 64000000 // (B * n))), n, dtype, residual, 0, codes,
                 weight)


# -------------------------------------------------------------------------------------- inputs
def _dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _randn(shape, case, gen, size=1.0):
    return (size * torch.randn(shape, generator=gen, device="cuda")).to(_dtype(case))


def _planes(x, case):
    """(B, H, N, D) or (B, N, H, D) as fp32 planes (B H, N, D)."""
    x = x if case["layout"] == "HND" else x.transpose(1, 2)
    return x.float().flatten(0, 1).contiguous()


def _back(x, case, H):
    """fp32 planes (B H, N, D) as (B, H, N, D) or (B, N, H, D)."""
    x = x.unflatten(0, (case["B"], H))
    x = x if case["layout"] == "HND" else x.transpose(1, 2)
    return x.to(_dtype(case)).contiguous()


def _groups(case):
    """Runs of query planes whose score matrices together hold about 2^30 values, and their K/V
    planes."""
    total, group = case["B"] * case["H"], case["H"] // case["H_kv"]
    at_once = max(1, (1 << 30) // (case["N"] * case["N_kv"]))
    for at in range(0, total, at_once):
        planes = torch.arange(at, min(at + at_once, total), device="cuda")
        yield planes, planes // group


def _scores(case, q, k):
    """Scores of planes q (P, N, D) on k (P, N_kv, D), masked."""
    s = (q * case["D"] ** -0.5) @ k.transpose(1, 2).contiguous()
    if case["causal"]:
        unseen = torch.ones(case["N"], case["N_kv"], dtype=torch.bool, device="cuda").triu(1)
        s.masked_fill_(unseen, -torch.inf)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "grad":
        B, H, H_kv, N, N_kv, D = (case[x] for x in ("B", "H", "H_kv", "N", "N_kv", "D"))

        def shape(h, n):
            return (B, h, n, D) if case["layout"] == "HND" else (B, n, h, D)
        # scores with a spread of 2, as of heads that look at some tokens more than at others
        state["q"] = _randn(shape(H, N), case, gen, 2.0)
        state["k"] = _randn(shape(H_kv, N_kv), case, gen)
        state["v"] = _randn(shape(H_kv, N_kv), case, gen)
        # a gradient's size, some way over fp16's least numbers
        state["dout"] = _randn(shape(H, N), case, gen, 2.0 ** -7)
        state["dlse"] = 2.0 ** -7 * torch.randn(B, H, N, generator=gen, device="cuda") \
            if case["dlse"] else None
        # what the forward call returned
        q, k, v = (_planes(state[x], case) for x in "qkv")
        out = torch.empty(B * H, N, D, device="cuda")
        lse = torch.empty(B * H, N, device="cuda")
        for planes, kv in _groups(case):
            s = _scores(case, q[planes], k[kv])
            top = s.amax(-1, keepdim=True)
            s.sub_(top).exp_()
            total = s.sum(-1, keepdim=True)
            out[planes] = s @ v[kv] / total
            lse[planes] = (top + total.log()).squeeze(-1)
            del s
        state["out"], state["lse"] = _back(out, case, H), lse.view(B, H, N)
        return state
    B, N, H, n = (case[x] for x in ("B", "N", "H", "n"))
    shape = (B, N, H, n) if H else (B, N, n)

    def rows():
        # rows whose sizes differ, with a few large columns, as a residual stream's
        x = torch.randn((B, N, 3 * H, n) if H else shape, generator=gen, device="cuda")
        x *= torch.rand(x.shape[:-1] + (1,), generator=gen, device="cuda") + 0.25
        x[..., ::max(n // 4, 1)] *= 8.0
        x = x.to(_dtype(case))
        return x[:, :, :H] if H else x
    state["x"] = rows()
    weight = 1.0 + 0.25 * torch.randn(n, generator=gen, device="cuda")
    state["weight"] = weight if case["weight"] == "fp32" else weight.to(_dtype(case))
    if case["op"] == "norm_grad":
        state["dy"] = _randn(shape, case, gen, 2.0 ** -7)
        state["dsum"] = _randn(shape, case, gen, 2.0 ** -7) if case["residual"] else None
        state["rstd"] = (state["x"].float().square().mean(-1) + EPS).rsqrt()
    else:
        state["residual"] = rows() if case["residual"] else None
    return state


# ---------------------------------------------------------------------------- the plain forms
def _plain_grad(state):
    case = state["case"]
    B, H, H_kv, N, N_kv, D = (case[x] for x in ("B", "H", "H_kv", "N", "N_kv", "D"))
    q, k, v, out, dout = (_planes(state[x], case) for x in ("q", "k", "v", "out", "dout"))
    lse = state["lse"].reshape(B * H, N, 1)
    drop = (dout * out).sum(-1, keepdim=True)
    if case["dlse"]:
        drop = drop - state["dlse"].reshape(B * H, N, 1)
    dq = torch.empty(B * H, N, D, device="cuda")
    dk = torch.zeros(B * H_kv, N_kv, D, device="cuda")
    dv = torch.zeros(B * H_kv, N_kv, D, device="cuda")
    for planes, kv in _groups(case):
        p = _scores(case, q[planes], k[kv]).sub_(lse[planes]).exp_()
        dv.index_add_(0, kv, p.transpose(1, 2).contiguous() @ dout[planes])
        ds = dout[planes] @ v[kv].transpose(1, 2).contiguous()
        ds.sub_(drop[planes]).mul_(p).mul_(D ** -0.5)
        del p
        dq[planes] = ds @ k[kv]
        dk.index_add_(0, kv, ds.transpose(1, 2).contiguous() @ q[planes])
        del ds
    return {"dq": _back(dq, case, H), "dk": _back(dk, case, H_kv), "dv": _back(dv, case, H_kv)}


def _quantize(y, codes):
    """Codes and scales of fp32 rows."""
    most = torch.full((), 127.0 if codes == "int8" else 448.0, device=y.device)
    scale = (y.abs().amax(-1) / most).clamp(min=FLOOR)
    code = y / scale[..., None]
    if codes == "int8":
        return code.round().clamp(-128, 127).to(torch.int8), scale
    return code.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _values(codes, scales):
    """What the codes stand for: int8 ones times their scale; e4m3 ones are values."""
    return codes * scales[..., None] if codes.dtype == torch.int8 else codes


def _plain_norm(state):
    case, dtype = state["case"], _dtype(state["case"])
    x = state["x"].float()
    if case["residual"]:
        x = x + state["residual"].float()
    y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * state["weight"].float()
    done = {"sum": x.to(dtype)} if case["residual"] else {}
    if case["op"] == "quant":
        codes, scales = _quantize(y, case["codes"])
        return dict(done, y=_values(codes, scales), scales=scales)
    return dict(done, y=y.to(dtype))


def _plain_norm_grad(state):
    x, dy, rstd = state["x"].float(), state["dy"].float(), state["rstd"][..., None]
    xhat = x * rstd
    g = dy * state["weight"].float()
    dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    if state["dsum"] is not None:
        dx = dx + state["dsum"].float()
    dw = (dy * xhat).flatten(0, -2).sum(0)
    return {"dx": dx.to(state["x"].dtype), "dw": dw.to(state["weight"].dtype)}


# ------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _own(state)
    if case["op"] == "grad":
        return _plain_grad(state)
    return _plain_norm_grad(state) if case["op"] == "norm_grad" else _plain_norm(state)


def _own(state):
    import sageattention as sage
    case = state["case"]
    if case["op"] == "grad":
        dq, dk, dv = sage.sageattn_backward(
            state["dout"], state["q"], state["k"], state["v"], state["out"], state["lse"],
            tensor_layout=case["layout"], is_causal=case["causal"], dlse=state["dlse"])
        return {"dq": dq, "dk": dk, "dv": dv}
    if case["op"] == "norm_grad":
        dx, dw = sage.rms_norm_backward(state["dy"], state["x"], state["weight"], state["rstd"],
                                        dsum=state["dsum"])
        return {"dx": dx, "dw": dw}
    if case["op"] == "quant":
        made = sage.rms_norm_quant(state["x"], state["weight"], EPS, residual=state["residual"],
                                   int8=case["codes"] == "int8")
        done = {"y": _values(made[0], made[1]), "scales": made[1]}
        return dict(done, sum=made[2]) if case["residual"] else done
    if case["residual"]:
        y, total = sage.rms_norm(state["x"], state["weight"], EPS, residual=state["residual"])
        return {"y": y, "sum": total}
    return {"y": sage.rms_norm(state["x"], state["weight"], EPS)}


# --------------------------------------------------------------------------- work and results
def work(case):
    if case["op"] == "grad":
        B, H, H_kv, N, N_kv, D = (case[x] for x in ("B", "H", "H_kv", "N", "N_kv", "D"))
        pairs = N * (N + 1) / 2 if case["causal"] else N * N_kv
        rows = B * H * N
        # q, out, dout in, dq out; k, v in, dk, dv out; the logsumexp and its gradient
        bytes_ = rows * (8 * D + 4 + 4 * case["dlse"]) + B * H_kv * N_kv * 8 * D
        return {"bytes": bytes_, "flops": 10 * B * H * pairs * D}   # five products
    rows = case["B"] * case["N"] * max(case["H"], 1)
    n, weight = case["n"], 4 if case["weight"] == "fp32" else 2
    if case["op"] == "norm_grad":
        bytes_ = rows * n * (8 if case["residual"] else 6) + 4 * rows + 2 * weight * n
        return {"bytes": bytes_, "flops": 9 * rows * n}
    made = rows * n * (1 if case["op"] == "quant" else 2) + (4 * rows if case["op"] == "quant" else 0)
    # codes of int8 come back as fp32 values
    made += rows * n * 5 if case["codes"] == "int8" else 0
    return {"bytes": rows * n * (6 if case["residual"] else 2) + made + weight * n,
            "flops": 5 * rows * n}


def exact(case, seed):
    """`run`'s result from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "grad":
        return _exact_grad(s)
    if case["op"] == "norm_grad":
        return _exact_norm_grad(s)
    t = s["x"].double()
    if s["residual"] is not None:
        t = t + s["residual"].double()
    size = torch.sqrt(torch.sum(t ** 2, -1) / case["n"] + EPS)
    y = t / size.unsqueeze(-1) * s["weight"].double()
    result = {}
    if s["residual"] is not None:
        result["sum"] = t
    if case["op"] == "norm":
        return dict(result, y=y)
    most = 127 if case["codes"] == "int8" else 448
    scales = torch.clamp(y.abs().max(-1).values / most, min=FLOOR)
    steps = y / scales.unsqueeze(-1)
    if case["codes"] == "int8":
        y = torch.round(steps) * scales.unsqueeze(-1)
    else:
        y = torch.clamp(steps, -448, 448).to(torch.float8_e4m3fn).double()
    return dict(result, y=y, scales=scales)


def _exact_norm_grad(s):
    """dx = (g - t (g . t) / (n size^2)) / size for g = dy weight, t the row and 1 / size = rstd."""
    n = s["case"]["n"]
    t, dy, r = s["x"].double(), s["dy"].double(), s["rstd"].double().unsqueeze(-1)
    g = dy * s["weight"].double()
    along = torch.sum(g * t, -1, keepdim=True)
    dx = g * r - t * along * r ** 3 / n
    if s["dsum"] is not None:
        dx = dx + s["dsum"].double()
    dw = torch.sum((dy * t * r).reshape(-1, n), 0)
    return {"dx": dx, "dw": dw}


def _exact_grad(s):
    """Head by head: for a row's weights p = exp(score - lse), the gradient of value j is the sum of
    p_j dout over the rows, that of score j is p_j (dout . v_j - dout . out + dlse)."""
    case = s["case"]
    B, H, H_kv, N, N_kv, D = (case[x] for x in ("B", "H", "H_kv", "N", "N_kv", "D"))

    def head(x, b, h):
        return (x[b, h] if case["layout"] == "HND" else x[b, :, h]).double()
    dq = torch.empty(B, H, N, D, dtype=torch.float64, device="cuda")
    dk = torch.zeros(B, H_kv, N_kv, D, dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    # a slice of rows at a time: 2^28 scores at most
    step = max(1, (1 << 28) // N_kv)
    column = torch.arange(N_kv, device="cuda")
    for b in range(B):
        for h in range(H):
            own_kv = h * H_kv // H
            keys, vals = head(s["k"], b, own_kv), head(s["v"], b, own_kv)
            keys_t, vals_t = keys.t().contiguous(), vals.t().contiguous()
            for at in range(0, N, step):
                to = min(at + step, N)
                # rows before `to` see no key behind it when causal
                m = to if case["causal"] else N_kv
                rows, grad = head(s["q"], b, h)[at:to], head(s["dout"], b, h)[at:to]
                p = torch.exp(torch.mm(rows, keys_t[:, :m]) / D ** 0.5
                              - s["lse"][b, h, at:to].double().unsqueeze(1))
                if case["causal"]:
                    row = torch.arange(at, to, device="cuda").unsqueeze(1)
                    p = torch.where(column[:m] <= row, p, torch.zeros_like(p))
                dv[b, own_kv, :m] += torch.mm(p.t().contiguous(), grad)
                less = torch.sum(grad * head(s["out"], b, h)[at:to], 1)
                if s["dlse"] is not None:
                    less = less - s["dlse"][b, h, at:to].double()
                p = p * (torch.mm(grad, vals_t[:, :m]) - less.unsqueeze(1)) / D ** 0.5
                dq[b, h, at:to] = torch.mm(p, keys[:m])
                dk[b, own_kv, :m] += torch.mm(p.t().contiguous(), rows)
    results = {"dq": dq, "dk": dk, "dv": dv}
    if case["layout"] == "HND":
        return results
    return {name: x.transpose(1, 2).contiguous() for name, x in results.items()}
