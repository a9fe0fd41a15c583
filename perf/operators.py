"""Serving from a quantized K/V cache: the operators' calls, their inputs, work and results.

Four operators, as one decoding step of a language model uses them next to `sageattn`:

* `rotary`: rotary positions applied to a query (or gradient) tensor, both pair layouts, on a part of
  the head, with an fp32 table of cosines and sines that holds any scaling for long contexts;
* `write`: new tokens' K and V quantized per token (K int8 or e4m3, V e4m3) into a paged cache, K
  rotated on the way; "write, then read" also reads the tokens back;
* `read`: cached tokens back in 16 bits;
* `attn`: attention of a sequence's newest tokens (one, or a tree of drafted ones with its mask) over
  all of its cached tokens.

`listed()` names the calls that stand for real use, `draw(rng)` gives others of the same ranges.
`run` computes the plain form in 32 bits, or, where `own` is true, calls the framework.
"""
import os
import sys

import torch

#: whether `run` calls the framework's operators
own = False

PAGE = 64            # tokens of a cache page
FLOOR = 1e-12        # the least row scale


# --------------------------------------------------------------------------------------- cases
def _rotary(B, H, N, D, R, dtype, layout, interleaved, inverse=False):
    return {"op": "rotary", "B": B, "H": H, "N": N, "D": D, "R": R, "dtype": dtype,
            "layout": layout, "interleaved": interleaved, "inverse": inverse}


def _write(B, H_kv, N, past, D, dtype, int8, layout, R, interleaved=False):
    return {"op": "write", "B": B, "H_kv": H_kv, "N": N, "past": past, "D": D, "dtype": dtype,
            "int8": int8, "layout": layout, "R": R, "interleaved": interleaved}


def _read(B, H_kv, L, D, dtype, int8, layout, ragged):
    return {"op": "read", "B": B, "H_kv": H_kv, "L": L, "D": D, "dtype": dtype, "int8": int8,
            "layout": layout, "ragged": ragged}


def _attn(B, H, H_kv, T, L, D, dtype, int8, layout="NHD", tree=False, ragged=False, lse=False):
    return {"op": "attn", "B": B, "H": H, "H_kv": H_kv, "T": T, "L": L, "D": D, "dtype": dtype,
            "int8": int8, "layout": layout, "tree": tree, "ragged": ragged, "lse": lse}


def listed():
    named = {
        # the queries of one decoding step of a batch: launch latency
        "rotary_step": _rotary(64, 32, 1, 128, 128, "bf16", "HND", False),
        # the queries of a long video, half of each head rotated in adjacent pairs
        "rotary_video": _rotary(1, 48, 47520, 128, 64, "fp16", "NHD", True),
        # one new token of each sequence of a batch, K rotated, into the pages that they fill
        "write_step": _write(128, 8, 1, 1000, 128, "bf16", False, "HND", 128),
        # prompts written and read back, so that their own attention sees what the cache holds
        "write_read_prompt": _write(4, 8, 4001, 0, 128, "fp16", True, "NHD", 0),
        # short cached prefixes of a batch, read back for a prompt's second part
        "read_short": _read(8, 10, 700, 64, "fp16", True, "HND", True),
        # one long cached document
        "read_long": _read(1, 8, 32768, 128, "bf16", False, "NHD", False),
        # one user's next token early in a conversation: latency
        "decode_one": _attn(1, 32, 8, 1, 517, 128, "fp16", True),
        # a serving batch's next tokens, lengths spread up to 8192
        "decode_batch": _attn(64, 32, 8, 1, 8192, 128, "bf16", False, ragged=True),
        # a few long documents, with the logsumexp that merges other keys' attention in
        "decode_long": _attn(4, 48, 8, 1, 131072, 128, "fp16", True, lse=True),
        # a small tree drafted for two sequences, as many K/V heads as heads, head_dim 64
        "tree_small": _attn(2, 10, 10, 7, 1024, 64, "fp16", True, layout="HND", tree=True),
        # trees of 33 drafted tokens for a batch of ragged sequences
        "tree_batch": _attn(16, 32, 8, 33, 4096, 128, "bf16", False, tree=True, ragged=True),
        # wide trees over long contexts: products matter as much as the cache's bytes
        "tree_wide": _attn(8, 32, 4, 64, 32768, 128, "fp16", True, tree=True),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("rotary", "write", "read", "attn", "attn", "attn"))
    D = rng.choice((128, 128, 64))
    layout = rng.choice(("HND", "NHD"))
    dtype = rng.choice(("fp16", "bf16"))
    int8 = dtype == "fp16" and rng.random() < 0.7
    if op == "rotary":
        H, B = rng.choice((8, 10, 32, 48)), _size(rng, 1, 64)
        N = _size(rng, 1, max(1, 2000000 // (B * H)))
        return _rotary(B, H, N, D, rng.choice((D, D, D // 2, D // 4)), dtype, layout,
                       rng.random() < 0.5, rng.random() < 0.3)
    H_kv = rng.choice((1, 2, 4, 8, 10))
    if op == "write":
        B = _size(rng, 1, 128)
        return _write(B, H_kv, _size(rng, 1, max(1, 16000 // B)), _size(rng, 1, 1000), D, dtype,
                      int8, layout, rng.choice((0, D, D // 2)), rng.random() < 0.5)
    if op == "read":
        B = _size(rng, 1, 16)
        return _read(B, H_kv, _size(rng, 1, max(64, 32768 // B)), D, dtype, int8, layout,
                     rng.random() < 0.5)
    tree = rng.random() < 0.6
    T = _size(rng, 2, 128) if tree else rng.choice((1, 1, 2, 5))
    H = H_kv * rng.choice((1, 4, 6, 8))
    B = _size(rng, 1, 64)
    # at most the queries times keys of the listed cases with the most of them
    most = min(131072, 8 * 32 * 64 * 32768 // (B * H * T), 4 * 8 * 131072 // (B * H_kv))
    return _attn(B, H, H_kv, T, max(T, _size(rng, 16, max(17, most))), D, dtype, int8, layout,
                 tree, rng.random() < 0.5, rng.random() < 0.3)


def _lens(case):
    """Each sequence's cached tokens: all alike, or spread evenly up to the longest."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    return [max(case.get("T", 1), L * (b + 1) // B - b % 3) for b in range(B)]


# -------------------------------------------------------------------------------------- inputs
def _dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _randn(shape, case, gen, layout):
    """Unit normal (B, H, N, D), or (B, N, H, D) for the layout NHD."""
    B, H, N, D = shape
    shape = (B, H, N, D) if layout == "HND" else (B, N, H, D)
    return torch.randn(shape, generator=gen, device="cuda").to(_dtype(case))


def _table(rows, R):
    """fp32 (rows, R): the cosines of R/2 frequencies, then their sines, worked out in 64 bits;
    positions stretched by two, as for a context twice as long as the trained one."""
    freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] / 2.0 * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _pool(case, pages, gen):
    """A cache's pages: codes and scales as quantized unit normal rows have them."""
    shape = (pages, case["H_kv"], PAGE, case["D"])
    k = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    k8 = (k * 40).round().clamp(-127, 127).to(torch.int8) if case["int8"] else \
        (k * 150).clamp(-448, 448).to(torch.float8_e4m3fn)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    v8 = (v * 150).clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = torch.rand((2,) + shape[:3], generator=gen, device="cuda") + 0.5
    return {"k8": k8, "sk": scale[0] / (40 if case["int8"] else 150), "v8": v8, "sv": scale[1] / 150}


def _tables(lens, pages, gen):
    """Each sequence's pages, in no order; rows are padded with -1, as nothing lies there."""
    width = max(-(-n // PAGE) for n in lens)
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    rows, at = [], 0
    for n in lens:
        used = -(-n // PAGE)
        rows.append(torch.cat((order[at:at + used], order.new_full((width - used,), -1))))
        at += used
    return torch.stack(rows)


def _tree(B, T, rng):
    """Masks of random trees: token j's parent is an earlier one, or the context; a token sees
    itself and its ancestors."""
    masks = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for j in range(T):
            up = int(torch.randint(-1, max(j, 1), (1,), generator=rng)) if j else -1
            if up >= 0:
                masks[b, j] = masks[b, up]
            masks[b, j, j] = True
    return masks.cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "rotary":
        B, N = case["B"], case["N"]
        state["x"] = _randn((B, case["H"], N, case["D"]), case, gen, case["layout"])
        state["table"] = _table(N + 4096, case["R"])
        start = torch.randint(0, 4096, (B, 1), generator=gen, device="cuda")
        state["positions"] = (start + torch.arange(N, device="cuda")).int()
        return state
    if case["op"] == "write":
        B, N = case["B"], case["N"]
        past = [max(0, case["past"] - 7 * (b % 5)) for b in range(B)]
        lens = [n + N for n in past]
        shape = (B, case["H_kv"], N, case["D"])
        state["k"] = _randn(shape, case, gen, case["layout"])
        state["v"] = _randn(shape, case, gen, case["layout"])
        state["start"] = torch.tensor(past, dtype=torch.int32, device="cuda")
        state["new"] = torch.full((B,), N, dtype=torch.int32, device="cuda")
        state["table"] = state["positions"] = None
        if case["R"]:
            state["table"] = _table(max(lens), case["R"])
            state["positions"] = state["start"][:, None] + \
                torch.arange(N, dtype=torch.int32, device="cuda")
    else:
        lens = _lens(case)
        state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pages = sum(-(-n // PAGE) for n in lens) + 1
    state["pool"] = _pool(case, pages, gen)
    state["pages"] = _tables(lens, pages, gen)
    if case["op"] == "attn":
        shape = (case["B"], case["H"], case["T"], case["D"])
        # scores with a spread of 3, as of heads that look at some tokens more than at others
        state["q"] = 3 * _randn(shape, case, gen, case["layout"])
        state["mask"] = _tree(case["B"], case["T"], torch.Generator().manual_seed(seed)) \
            if case["tree"] else None
    if own:
        # the handle that a serving program keeps over its pool of pages
        from sageattention import KVCache
        state["cache"] = KVCache(**state["pool"], dtype=_dtype(case))
    return state


# ---------------------------------------------------------------------------- the plain forms
def _rotate(x, table, positions, R, interleaved, inverse):
    """x (B, H, N, D) fp32 with its first R columns rotated."""
    cs = table[positions.long()][:, None]
    c, s = cs[..., :R // 2], cs[..., R // 2:]
    s = -s if inverse else s
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _quantize(x, most, int8):
    """Codes and scales of fp32 rows."""
    top = torch.full((), most, device=x.device)   # a tensor: division by a number multiplies
    scale = (x.abs().amax(-1) / top).clamp(min=FLOOR)
    code = x / scale[..., None]
    if int8:
        return code.round().clamp(-128, 127).to(torch.int8), scale
    return code.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _hnd(x, case):
    return x if case["layout"] == "HND" else x.transpose(1, 2)


def _gather(pool, pages, codes, scales):
    """The sequences' rows (B, H, width * PAGE, D) in fp32."""
    at = pages.long().clamp(min=0)
    rows = pool[codes].view(torch.uint8)[at].view(pool[codes].dtype).float()
    rows = rows * pool[scales][at][..., None]
    return rows.transpose(1, 2).flatten(2, 3)


def _plain_read(state, first, count):
    """Rows first[b] .. first[b] + count[b] - 1 of each sequence, as many as the longest."""
    case = state["case"]
    n = case["N"] if case["op"] == "write" else case["L"]
    at = first.long()[:, None] + torch.arange(n, device="cuda")
    live = torch.arange(n, device="cuda") < count[:, None]
    at = at.clamp(max=state["pages"].shape[1] * PAGE - 1)
    page = state["pages"].long().gather(1, at // PAGE).clamp(min=0)
    out = []
    for codes, scales in (("k8", "sk"), ("v8", "sv")):
        pool = state["pool"][codes]
        rows = pool.view(torch.uint8)[page, :, at % PAGE].view(pool.dtype).float()
        rows = rows * state["pool"][scales][page, :, at % PAGE][..., None]
        rows = (rows * live[..., None, None]).to(_dtype(case))
        out.append(rows.transpose(1, 2).contiguous() if case["layout"] == "HND" else rows)
    return out


def _plain_write(state):
    case, pool = state["case"], state["pool"]
    k, v = _hnd(state["k"], case).float(), _hnd(state["v"], case).float()
    if case["R"]:
        k = _rotate(k, state["table"], state["positions"], case["R"], case["interleaved"], False)
    at = state["start"].long()[:, None] + torch.arange(case["N"], device="cuda")
    page = state["pages"].long().gather(1, at // PAGE)
    for x, most, int8, codes, scales in (
            (k, 127.0 if case["int8"] else 448.0, case["int8"], "k8", "sk"),
            (v, 448.0, False, "v8", "sv")):
        code, scale = _quantize(x, most, int8)
        pool[codes].view(torch.uint8)[page, :, at % PAGE] = code.view(torch.uint8).transpose(1, 2)
        pool[scales][page, :, at % PAGE] = scale.transpose(1, 2)


def _seen(state):
    """(B, T, keys): which cached tokens each new token sees."""
    case, T = state["case"], state["case"]["T"]
    key = torch.arange(state["pages"].shape[1] * PAGE, device="cuda")
    lens = state["lens"].long()[:, None, None]
    draft = key - (lens - T)                       # the key's place among the new tokens
    if state["mask"] is None:
        within = draft <= torch.arange(T, device="cuda")[:, None]
    else:
        at = draft.clamp(0, T - 1).expand(-1, T, -1)
        within = state["mask"].gather(2, at) | (draft < 0)
    return within & (key < lens)


def _plain_attn(state):
    case = state["case"]
    B, H, H_kv, T, D = (case[n] for n in ("B", "H", "H_kv", "T", "D"))
    q = _hnd(state["q"], case).float().reshape(B, H_kv, H // H_kv * T, D)
    k = _gather(state["pool"], state["pages"], "k8", "sk")
    s = (q * D ** -0.5) @ k.transpose(2, 3).contiguous()
    del k
    seen = _seen(state)[:, None, None]
    s = s.view(B, H_kv, H // H_kv, T, -1).masked_fill_(~seen, -torch.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(B, H_kv, H // H_kv * T, -1) @ _gather(state["pool"], state["pages"], "v8", "sv")
    o = o.view(B, H_kv, H // H_kv, T, D) / total.clamp(min=1e-30)
    o = o.reshape(B, H, T, D).to(_dtype(case))
    o = o if case["layout"] == "HND" else o.transpose(1, 2).contiguous()
    return (o, (top + total.log()).view(B, H, T)) if case["lse"] else o


# ------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _own(state)
    if case["op"] == "rotary":
        x = _hnd(state["x"], case).float()
        y = _rotate(x, state["table"], state["positions"], case["R"], case["interleaved"],
                    case["inverse"])
        return _hnd(y, case).to(_dtype(case)).contiguous()
    if case["op"] == "write":
        _plain_write(state)
        # int8 codes are read back as the values they stand for; e4m3 codes are values
        return _plain_read(state, state["start"], state["new"]) if case["int8"] else state["pool"]
    if case["op"] == "read":
        return _plain_read(state, torch.zeros_like(state["lens"]), state["lens"])
    return _plain_attn(state)


def _own(state):
    from sageattention import apply_rotary, sageattn_cached
    case = state["case"]
    if case["op"] == "rotary":
        return apply_rotary(state["x"], state["table"], state["positions"],
                            tensor_layout=case["layout"], interleaved=case["interleaved"],
                            inverse=case["inverse"])
    cache = state["cache"]
    if case["op"] == "write":
        cache.write(state["k"], state["v"], state["pages"], state["start"],
                    tensor_layout=case["layout"], table=state["table"],
                    positions=state["positions"], interleaved=case["interleaved"])
        return cache.read(state["pages"], state["new"], case["N"], start=state["start"],
                          tensor_layout=case["layout"]) if case["int8"] else state["pool"]
    if case["op"] == "read":
        return cache.read(state["pages"], state["lens"], case["L"], tensor_layout=case["layout"])
    return sageattn_cached(state["q"], cache, state["pages"], state["lens"],
                           tensor_layout=case["layout"], tree_mask=state["mask"],
                           return_lse=case["lse"])


# --------------------------------------------------------------------------- work and results
def work(case):
    D = case["D"]
    if case["op"] == "rotary":
        rows = case["B"] * case["H"] * case["N"]
        # each row in and out; a token's cosines and sines and its position
        return {"bytes": rows * D * 4 + case["B"] * case["N"] * (case["R"] * 4 + 4),
                "flops": 3 * rows * case["R"]}
    held = 2 * D + 8                   # a token's codes and scales of one head, K and V
    if case["op"] == "write":
        rows = case["B"] * case["H_kv"] * case["N"]
        bytes_ = rows * (4 * D + held) + case["B"] * case["N"] * 4 * case["R"]
        return {"bytes": bytes_ + (rows * (held + 4 * D) if case["int8"] else 0),
                "flops": rows * D * (8 if case["int8"] else 6)}
    tokens = sum(_lens(case))
    if case["op"] == "read":
        return {"bytes": case["H_kv"] * (tokens * held + case["B"] * case["L"] * 4 * D),
                "flops": 2 * case["H_kv"] * tokens * D}
    rows = case["B"] * case["H"] * case["T"]
    return {"bytes": case["H_kv"] * tokens * held + rows * 4 * D + (4 * rows if case["lse"] else 0),
            "flops": 4 * case["H"] * case["T"] * tokens * D}


def exact(case, seed):
    """`run`'s result from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_turn(s["x"].double(), s, case["layout"] == "HND",
                           -1.0 if case["inverse"] else 1.0)
    if case["op"] == "read":
        return _exact_rows(s, lambda b: range(int(s["lens"][b])), case["L"])
    if case["op"] == "write":
        return _exact_write(s)
    return _exact_attn(s)


def _exact_turn(x, s, heads_first, sign):
    """Each pair (a, b) as the complex number a + ib, times the position's unit number."""
    case, R = s["case"], s["case"]["R"]
    cs = s["table"].double()[s["positions"].long()]
    turn = torch.complex(cs[..., :R // 2], sign * cs[..., R // 2:])
    turn = turn.unsqueeze(1 if heads_first else 2)
    y = x.clone()
    lo, hi = (slice(0, R, 2), slice(1, R, 2)) if case["interleaved"] else \
        (slice(0, R // 2), slice(R // 2, R))
    z = torch.complex(x[..., lo].contiguous(), x[..., hi].contiguous()) * turn
    y[..., lo], y[..., hi] = z.real, z.imag
    return y


def _exact_values(s, b, places, codes, scales):
    """Sequence b's rows at these places: (H_kv, places, D)."""
    at = torch.tensor(list(places), device="cuda")
    page, slot = s["pages"][b].long()[at // PAGE], at % PAGE
    rows = s["pool"][codes].view(torch.uint8)[page, :, slot].view(s["pool"][codes].dtype).double()
    return (rows * s["pool"][scales].double()[page, :, slot][..., None]).transpose(0, 1)


def _exact_rows(s, places, n):
    case, out = s["case"], []
    for codes, scales in (("k8", "sk"), ("v8", "sv")):
        y = torch.zeros(case["B"], case["H_kv"], n, case["D"], dtype=torch.float64, device="cuda")
        for b in range(case["B"]):
            at = places(b)
            y[b, :, :len(at)] = _exact_values(s, b, at, codes, scales)
        out.append(y if case["layout"] == "HND" else y.transpose(1, 2).contiguous())
    return out


def _exact_write(s):
    case = s["case"]
    k, v = s["k"].double(), s["v"].double()
    if case["R"]:
        k = _exact_turn(k, s, case["layout"] == "HND", 1.0)
    k, v = (x if case["layout"] == "NHD" else x.transpose(1, 2) for x in (k, v))
    at = s["start"].long()[:, None] + torch.arange(case["N"], device="cuda")
    page = torch.gather(s["pages"].long(), 1, at // PAGE)
    held, back = {}, []
    for name, x, most in (("k", k, 127 if case["int8"] else 448), ("v", v, 448)):
        scale = torch.clamp(x.abs().max(-1).values / most, min=FLOOR)
        steps = x / scale.unsqueeze(-1)
        steps = torch.round(steps) if most == 127 else \
            steps.clamp(-448, 448).to(torch.float8_e4m3fn).double()
        back.append(steps * scale.unsqueeze(-1))
        codes, scales = s["pool"][name + "8"].double(), s["pool"]["s" + name].double()
        codes[page, :, at % PAGE], scales[page, :, at % PAGE] = steps, scale
        held[name + "8"], held["s" + name] = codes, scales
    if not case["int8"]:
        return held
    return [x if case["layout"] == "NHD" else x.transpose(1, 2).contiguous() for x in back]


def _exact_attn(s):
    case = s["case"]
    H, H_kv, T, D = (case[n] for n in ("H", "H_kv", "T", "D"))
    q = s["q"].double() if case["layout"] == "HND" else s["q"].double().transpose(1, 2)
    outs, sums = [], []
    for b, n in enumerate(_lens(case)):
        k, v = (_exact_values(s, b, range(n), *names) for names in (("k8", "sk"), ("v8", "sv")))
        # new token i sees the n - T tokens before the tree, and those of the tree that it may
        tree = torch.ones(T, T, dtype=torch.bool, device="cuda").tril() if s["mask"] is None \
            else s["mask"][b]
        for h in range(H):
            score = q[b, h] @ k[h * H_kv // H].T.contiguous() / D ** 0.5
            score[:, n - T:][~tree] = -torch.inf
            sums.append(torch.logsumexp(score, 1))
            outs.append(torch.softmax(score, 1) @ v[h * H_kv // H])
    o = torch.stack(outs).view(case["B"], H, T, D)
    o = o if case["layout"] == "HND" else o.transpose(1, 2).contiguous()
    return (o, torch.stack(sums).view(case["B"], H, T)) if case["lse"] else o


if not any(p.endswith("sageattention-rdna4_amd") for p in sys.path):
    sys.path.insert(0, os.path.join(os.getcwd(), "sageattention-rdna4_amd"))
