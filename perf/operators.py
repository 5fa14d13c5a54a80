"""Cases of the token-order and 8-bit operators: what is measured, and their plain forms.

    dispatch   token-expert pairs sorted by expert, and the token rows gathered in that order
    combine    expert rows back to their tokens, weighted and summed in rank order
    backward   the gradients of both: of the expert rows and of the weights (combine), of the tokens (gather)
    linear     a dense product in 8-bit integers: rows quantised per token, weights per output channel
    experts    the same product with one weight matrix per expert over rows in expert order; gate_up takes the
               tokens themselves (gathered while they are quantised) and applies SwiGLU, down takes expert rows

Sizes are those of the layers that the benchmark runs (hidden 2048 or 1024, 128 or 16 experts, expert width 768
or 512, q projection 2048 -> 4096), and odd ones.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a decode step of eight sequences: latency
        {"name": "dispatch_decode", "op": "dispatch", "T": 8, "H": 2048, "E": 128, "k": 8, "x": "f32", "y": "bf16",
         "skew": 0.0, "pad": 0.0},
        # a prompt chunk whose router load is skewed, as the prefill benchmark's
        {"name": "dispatch_prefill", "op": "dispatch", "T": 4096, "H": 2048, "E": 128, "k": 8, "x": "bf16", "y": "bf16",
         "skew": 1.1, "pad": 0.0},
        # a decode batch of the small 16-expert layer, f32 as its forward keeps its rows
        {"name": "combine_decode", "op": "combine", "T": 32, "H": 1024, "E": 16, "k": 4, "x": "f32", "y": "f32",
         "skew": 0.0, "pad": 0.0},
        {"name": "combine_prefill", "op": "combine", "T": 4096, "H": 2048, "E": 128, "k": 8, "x": "bf16", "y": "f32",
         "skew": 1.1, "pad": 0.0},
        # a ragged training batch with padding tokens that no expert takes
        {"name": "backward_ragged", "op": "backward", "T": 333, "H": 1000, "E": 60, "k": 6, "x": "f32", "y": "f32",
         "skew": 0.5, "pad": 0.1},
        {"name": "backward_prefill", "op": "backward", "T": 4096, "H": 2048, "E": 128, "k": 8, "x": "bf16", "y": "bf16",
         "skew": 1.1, "pad": 0.0},
        # the q projection of one decoded token
        {"name": "linear_token", "op": "linear", "T": 1, "K": 2048, "O": 4096, "x": "f32", "y": "f32"},
        {"name": "linear_ragged", "op": "linear", "T": 77, "K": 1000, "O": 1500, "x": "f16", "y": "f32"},
        {"name": "linear_prefill", "op": "linear", "T": 4096, "K": 2048, "O": 4096, "x": "bf16", "y": "bf16"},
        # decode batch: nearly every expert's weights are read for a few rows each
        {"name": "gate_up_decode", "op": "gate_up", "T": 64, "H": 2048, "E": 128, "k": 8, "I": 768, "x": "f32", "y": "f32",
         "skew": 0.0, "pad": 0.0},
        {"name": "gate_up_prefill", "op": "gate_up", "T": 4096, "H": 2048, "E": 128, "k": 8, "I": 768, "x": "bf16",
         "y": "bf16", "skew": 1.1, "pad": 0.0},
        # a short prompt: some dozens of rows for each expert
        {"name": "down_chunk", "op": "down", "T": 512, "H": 2048, "E": 128, "k": 8, "I": 768, "x": "bf16", "y": "bf16",
         "skew": 0.0, "pad": 0.0},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, evenly spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["dispatch", "combine", "backward", "linear", "gate_up", "down"])
    x, y = rng.choice(list(DTYPES)), rng.choice(list(DTYPES))
    if op == "linear":
        return {"op": op, "T": _spread(rng, 1, 4096), "K": _spread(rng, 32, 2048), "O": _spread(rng, 32, 4096), "x": x, "y": y}
    E = _spread(rng, 2, 128)
    case = {"op": op, "T": _spread(rng, 1, 4096), "H": _spread(rng, 32, 2048), "E": E, "k": rng.randint(1, min(8, E)),
            "x": x, "y": y, "skew": rng.choice([0.0, 0.5, 1.1]), "pad": rng.choice([0.0, 0.0, 0.1, 0.5])}
    if op in ("gate_up", "down"):
        case["I"] = _spread(rng, 16, 768)
    return case


# ---- inputs -------------------------------------------------------------------
def _routing(case, gen):
    """Selected experts [T, k] (distinct within a token, a power law of exponent `skew` over the experts; a share `pad` of
    the tokens is padding, marked -1) and their renormalised weights."""
    T, E, k = case["T"], case["E"], case["k"]
    bias = -case["skew"] * torch.log(torch.arange(1, E + 1, device=DEV, dtype=torch.float32))
    logits = bias + torch.randn(T, E, device=DEV, generator=gen)
    w, idx = torch.topk(torch.softmax(logits, 1), k, dim=1)
    idx = idx.to(torch.int32)
    if case["pad"]:
        idx[torch.rand(T, device=DEV, generator=gen) < case["pad"]] = -1
    return idx.contiguous(), (w / w.sum(1, keepdim=True)).contiguous()


def _rows(shape, dtype, gen):
    return torch.randn(shape, device=DEV, generator=gen).to(DTYPES[dtype])


def _codes(groups, out, width, gen):
    """8-bit weights with a scale for each output channel: rows of a normal matrix of deviation 0.02, quantised."""
    q = torch.empty((groups, out, width), dtype=torch.int8, device=DEV)
    scale = torch.empty((groups, out), dtype=torch.float32, device=DEV)
    step = max(1, (1 << 27) // (out * width))
    for g in range(0, groups, step):
        n = min(step, groups - g)
        w = torch.randn((n, out, width), device=DEV, generator=gen).mul_(0.02)
        s = w.abs().amax(2).div_(127).clamp_(min=1e-8)
        scale[g:g + n] = s
        q[g:g + n] = w.div_(s[:, :, None]).round_().clamp_(-127, 127).to(torch.int8)
    return q, scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op = case["op"]
    s = {"op": op, "case": case, "y": DTYPES[case["y"]]}
    if own:
        s["qg"] = _qgmoe()
    if op == "linear":
        s["x"] = _rows((case["T"], case["K"]), case["x"], gen)
        q, scale = _codes(1, case["O"], case["K"], gen)
        s["q"], s["scale"] = q, scale
        if own:
            s["lin"] = s["qg"].Int8Linear(q[0], scale[0])
        return s
    T, H, E, k = case["T"], case["H"], case["E"], case["k"]
    s["idx"], s["w"] = _routing(case, gen)
    if own:
        s["plan"] = s["qg"].TokenOrder(T, k, E)
        if op != "dispatch":
            s["plan"].sort(s["idx"])
    elif op != "dispatch":
        s["order"] = _plain_order(s["idx"], E)
    if op == "dispatch":
        s["x"] = _rows((T, H), case["x"], gen)
        s["rows"] = torch.zeros((T * k, H), dtype=s["y"], device=DEV)  # rows behind the last expert's stay as they are
    elif op == "combine":
        s["rows"] = _rows((T * k, H), case["x"], gen)
    elif op == "backward":
        s["rows"] = _rows((T * k, H), case["x"], gen)
        s["dout"] = _rows((T, H), case["y"], gen)
        s["drows"] = torch.zeros((T * k, H), dtype=s["rows"].dtype, device=DEV)
    elif op == "gate_up":
        s["x"] = _rows((T, H), case["x"], gen)
        s["q"], s["scale"] = _codes(E, 2 * case["I"], H, gen)
        s["out"] = torch.zeros((T * k, case["I"]), dtype=s["y"], device=DEV)
        if own:
            s["lin"] = s["qg"].Int8Linear(s["q"], s["scale"], swiglu=True)
    else:  # down: the rows are SwiGLU outputs, heavier at zero than a normal
        g = torch.randn((T * k, case["I"]), device=DEV, generator=gen)
        u = torch.randn((T * k, case["I"]), device=DEV, generator=gen)
        s["x"] = (g * torch.sigmoid(g) * u).to(DTYPES[case["x"]])
        s["q"], s["scale"] = _codes(E, H, case["I"], gen)
        s["out"] = torch.zeros((T * k, H), dtype=s["y"], device=DEV)
        if own:
            s["lin"] = s["qg"].Int8Linear(s["q"], s["scale"])
    return s


def _qgmoe():
    at = os.path.join(os.getcwd(), "qwen-go_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import qgmoe
    return qgmoe


# ---- plain forms ----------------------------------------------------------------
def _plain_order(idx, E):
    """(offsets [E + 1], pair_row [T, k], row_pair [T * k]): the pairs of each expert in their own order, experts ascending;
    -1 for a pair without an expert and for a row without a pair."""
    ids = idx.reshape(-1).long()
    N = ids.numel()
    valid = (ids >= 0) & (ids < E)
    hot = (ids[:, None] == torch.arange(E, device=ids.device)).to(torch.int32)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = hot.sum(0).cumsum(0)
    safe = ids.clamp(0, E - 1)
    rank = hot.cumsum(0).gather(1, safe[:, None])[:, 0] - 1
    pair_row = torch.where(valid, offsets[safe] + rank.to(torch.int32), -1).to(torch.int32)
    row_pair = torch.full((N + 1,), -1, dtype=torch.int32, device=ids.device)
    row_pair[torch.where(valid, pair_row.long(), N)] = torch.arange(N, dtype=torch.int32, device=ids.device)
    return offsets, pair_row.view(idx.shape), row_pair[:N]


def _plain_scatter(values, pair_row, rows):
    """`rows` [N, H] with values [T, k, H] at their pairs' rows; the other rows are left."""
    N, H = rows.shape
    to = torch.empty((N + 1, H), dtype=rows.dtype, device=rows.device)
    to[:N] = rows
    to[torch.where(pair_row < 0, N, pair_row).long().reshape(-1)] = values.reshape(N, H).to(rows.dtype)
    return to[:N]


def _plain_quantize(x):
    x = x.float()
    top = x.abs().amax(1)
    s = (top / torch.full_like(top, 127)).clamp(min=1e-8)  # a number as divisor would be multiplied by its inverse
    v = x / s[:, None]
    return (torch.sign(v) * torch.floor(v.abs() + 0.5)).clamp(-127, 127), s


def _plain_grouped(codes, s, slot, q, scale, T):
    """y [rows, out]: row r times the weights of expert slot[r] // T; slot is the row's own place among E * T."""
    E, out, width = q.shape
    at = torch.zeros((E * T + 1, width), device=codes.device)
    at[slot] = codes
    y = torch.bmm(at[:E * T].view(E, T, width), q.float().transpose(1, 2)).view(E * T, out)
    live = slot.clamp(max=E * T - 1)
    return y[live] * s[:, None] * scale[live // T]


def run(s):
    op = s["op"]
    if own:
        qg = s["qg"]
        if op == "dispatch":
            plan = s["plan"].sort(s["idx"])
            rows = qg.gather_rows(s["x"], plan, out=s["rows"])
            return plan.offsets, plan.pair_row, plan.row_pair, rows
        if op == "combine":
            return qg.combine_rows(s["rows"], s["w"], s["plan"], dtype=s["y"])
        if op == "backward":
            drows, dw = qg.combine_rows_backward(s["dout"], s["rows"], s["w"], s["plan"], grad_rows=s["drows"])
            return drows, dw, qg.gather_rows_backward(s["rows"], s["plan"], dtype=s["y"])
        if op == "linear":
            return s["lin"].forward_device(s["x"], dtype=s["y"])
        if op == "gate_up":
            return s["lin"].forward_device(s["x"], s["out"], order=s["plan"])
        return s["lin"].forward_device(s["x"], s["out"], offsets=s["plan"].offsets)

    case, y = s["case"], s["y"]
    if op == "linear":
        codes, sc = _plain_quantize(s["x"])
        return (torch.matmul(codes, s["q"][0].float().t()) * sc[:, None] * s["scale"][0]).to(y)
    if op == "dispatch":
        offsets, pair_row, row_pair = _plain_order(s["idx"], case["E"])
        x = s["x"][:, None, :].expand(-1, case["k"], -1)
        return offsets, pair_row, row_pair, _plain_scatter(x, pair_row, torch.zeros_like(s["rows"]))
    T, E, k = case["T"], case["E"], case["k"]
    offsets, pair_row, row_pair = s["order"]
    live = (pair_row >= 0)[:, :, None]
    if op == "combine":
        r = torch.where(live, s["rows"][pair_row.clamp(min=0).long()].float(), 0.0)
        return (r * s["w"][:, :, None]).sum(1).to(y)
    if op == "backward":
        d = s["dout"].float()[:, None, :]
        r = torch.where(live, s["rows"][pair_row.clamp(min=0).long()].float(), 0.0)
        drows = _plain_scatter(d * s["w"][:, :, None], pair_row, torch.zeros_like(s["rows"]))
        return drows, (r * d).sum(2), r.sum(1).to(y)
    pair = row_pair.clamp(min=0).long()
    expert = s["idx"].reshape(-1)[pair].long()
    slot = torch.where(row_pair < 0, E * T, expert * T + pair // k)
    live = (row_pair >= 0)[:, None]
    if op == "gate_up":
        codes, sc = _plain_quantize(s["x"])
        v = _plain_grouped(codes[pair // k], sc[pair // k], slot, s["q"], s["scale"], T)
        g, u = v[:, :case["I"]], v[:, case["I"]:]
        return torch.where(live, g / (1 + torch.exp(-g)) * u, 0.0).to(y)
    codes, sc = _plain_quantize(s["x"])
    return torch.where(live, _plain_grouped(codes, sc, slot, s["q"], s["scale"], T), 0.0).to(y)


# ---- work -------------------------------------------------------------------------
def work(case):
    op, sx, sy = case["op"], SIZE[case["x"]], SIZE[case["y"]]
    T = case["T"]
    if op == "linear":
        K, O = case["K"], case["O"]
        return {"bytes": T * K * sx + O * K + 4 * O + T * O * sy, "flops": 2 * T * K * O}
    H, E, k = case["H"], case["E"], case["k"]
    N = round(T * (1 - case["pad"])) * k  # pairs that have an expert
    if op == "dispatch":
        return {"bytes": 12 * T * k + 4 * (E + 1) + T * H * sx + N * H * sy, "flops": 0}
    if op == "combine":
        return {"bytes": 8 * T * k + N * H * sx + T * H * sy, "flops": 2 * N * H}
    if op == "backward":  # rows once, their gradients once, both token-shaped arrays once
        return {"bytes": 12 * T * k + 2 * N * H * sx + 2 * T * H * sy, "flops": 4 * N * H}
    used = E * (1 - (1 - min(1.0, k / E)) ** T)  # experts that some token takes
    I = case["I"]
    if op == "gate_up":
        return {"bytes": 4 * T * k + T * H * sx + used * 2 * I * (H + 4) + N * I * sy, "flops": 4 * N * H * I}
    return {"bytes": N * I * sx + used * H * (I + 4) + N * H * sy, "flops": 2 * N * H * I}


# ---- 64 bits ------------------------------------------------------------------------
def _exact_quantize(x):
    """Codes and scales: the scale and each quotient are float32 by definition, the code is the nearest whole number to
    the quotient, halves away from zero."""
    x = x.double()
    s = (x.abs().max(1).values.div(127.0)).float().clamp(min=1e-8).double()
    v = (x / s[:, None]).float().double()
    return torch.copysign(torch.floor(v.abs() + 0.5), v).clamp(-127, 127), s


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        c, sc = _exact_quantize(s["x"])
        return (c @ s["q"][0].double().T) * sc[:, None] * s["scale"][0].double()
    T, E, k = case["T"], case["E"], case["k"]
    N = T * k
    ids = s["idx"].reshape(-1).cpu().tolist()
    members = [[] for _ in range(E)]
    for p, e in enumerate(ids):
        if 0 <= e < E:
            members[e].append(p)
    flat = torch.tensor([p for m in members for p in m], dtype=torch.long, device=DEV)  # the pair of each row
    token = flat // k
    M = flat.numel()
    if op == "dispatch":
        rows = torch.zeros((N, case["H"]), dtype=torch.float64, device=DEV)
        rows[:M] = s["x"].double()[token]
        return None, None, None, rows
    w = s["w"].double().reshape(-1)[flat][:, None]
    if op == "combine":
        out = torch.zeros((T, case["H"]), dtype=torch.float64, device=DEV)
        return out.index_add_(0, token, w * s["rows"][:M].double())
    if op == "backward":
        d, rows = s["dout"].double(), s["rows"][:M].double()
        drows = torch.zeros((N, case["H"]), dtype=torch.float64, device=DEV)
        drows[:M] = w * d[token]
        dw = torch.zeros(N, dtype=torch.float64, device=DEV)
        dw[flat] = (rows * d[token]).sum(1)
        dx = torch.zeros((T, case["H"]), dtype=torch.float64, device=DEV).index_add_(0, token, rows)
        return drows, dw.view(T, k), dx
    c, sc = _exact_quantize(s["x"])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for e, m in enumerate(members):
        if not m:
            continue
        here = slice(row, row + len(m))
        at = token[here] if op == "gate_up" else here
        v = (c[at] @ s["q"][e].double().T) * sc[at][:, None] * s["scale"][e].double()
        if op == "gate_up":
            g, u = v.chunk(2, 1)
            v = g * torch.sigmoid(g) * u
        out[here] = v
        row += len(m)
    return out
