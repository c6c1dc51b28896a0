"""The operators of the hybrid's linear-attention layers and of 4-bit projections, as measured cases.

Three layers in four of the hybrid backbone hold no keys and values but, per conversation and head, one
matrix: a linear attention with a decay for each head. Its operators, and the 4-bit projections around them:

* ``prologue``  causal depthwise convolution (width 4) + SiLU over the projected q | k | v channels of every
                new row, q and k normalized per head, the decays ``g = -exp(a_log) softplus(a + dt_bias)``
                and the write strengths ``beta = sigmoid(b)``; the last inputs kept per conversation
                (``linear_prologue``)
* ``attention`` S <- e^g S + k (beta (v - e^g S^T k))^T (``rule`` "delta") or S <- e^g S + k v^T ("sum"), then
                o = S^T q / sqrt(dk), row after row of each conversation; with ``gate`` the layer's output
                norm, rmsnorm(o) * weight * silu(z) (``linear_attention``)
* ``proj``      y = W x (+ resid) with W in 4 bits and one scale (and minimum) per group of weights, for a few
                rows x (``fused_mm`` / ``resid_mm`` with a ``FourBitWeight``)
* ``block``     a layer: in-projection, prologue, attention with its output norm, out-projection + residual
                (``linear_block``)

Everything is float32; states [slots, heads, dv, dk] and the convolution's last inputs [slots, 3, channels].
Where ``own`` is false a pass computes these in plain torch operations on the same tensors.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6
TAPS = 4
CHUNK = 64


# ---------------------------------------------------------------------------- the cases
def _attn(name, op, B, rows, Hk=16, Hv=48, dk=128, dv=128, ragged=1, **more):
    c = {"op": op, "B": B, "rows": rows, "Hk": Hk, "Hv": Hv, "dk": dk, "dv": dv, "ragged": ragged, "rule": "delta",
         "gate": True, "fresh": False}
    c.update(more)
    return dict(c, name=name) if name else c


def _proj(name, M, K, N0, N1=0, N2=0, group=128, mins=False, scales="f16", resid=False):
    c = {"op": "proj", "M": M, "K": K, "N0": N0, "N1": N1, "N2": N2, "group": group, "mins": mins, "scales": scales,
         "resid": resid}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one conversation: what a call costs
        _attn("prologue_b1", "prologue", 1, 1, Hv=32),
        # a long prompt of one new conversation
        _attn("prologue_prompt4096", "prologue", 1, 4096, fresh=True),
        # one token of one conversation, with the layer's gated norm: latency
        _attn("linear_b1", "attention", 1, 1, Hv=32),
        # one token of each of 64 conversations: the states' bytes
        _attn("linear_b64", "attention", 64, 1),
        # ragged prompts of several new users in one call, the gated norm behind
        _attn("linear_prompts_ragged", "attention", 6, 777, Hv=32, ragged=2, fresh=True),
        # one long prompt
        _attn("linear_prompt8192", "attention", 1, 8192, gate=False, fresh=True),
        # the plain sum with a constant decay for each head, small keys, going on from a state
        _attn("linear_sum2048", "attention", 2, 2048, Hk=16, Hv=16, dk=64, rule="sum", gate=False),
        # one token through an o_proj with its residual
        _proj("proj4_o_4096", 1, 4096, 4096, resid=True),
        # one token through the largest weight of a layer (gate | up), small groups with minima
        _proj("proj4_gate_up", 1, 4096, 12288, 12288, group=32, mins=True),
        # five drafted tokens of two conversations through a layer's in-projection
        _proj("proj4_in_rows10", 10, 4096, 10240, 6144, 96, group=64, scales="f32"),
        # a layer for one token of one conversation
        _attn("block_b1", "block", 1, 1, Hv=32, hidden=2048, group=128),
        # a layer for the five drafted tokens of three conversations
        _attn("block_verify5_b3", "block", 3, 5, hidden=4096, group=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    kind = rng.choice(["prologue", "attention", "attention", "attention", "proj", "proj", "block"])
    if kind == "proj":
        N0 = 16 * _log(rng, 8, 1024) + rng.choice([0, 0, rng.randint(1, 15)])
        resid = rng.random() < 0.4
        N1, N2 = (0, 0) if resid or rng.random() < 0.4 else (_log(rng, 16, 8192), _log(rng, 16, 1024))
        return _proj("", rng.choice([1, 1, rng.randint(2, 16)]), 128 * _log(rng, 4, 96), N0, N1, N2,
                     rng.choice([32, 64, 128]), rng.random() < 0.4, rng.choice(["f16", "f32"]), resid)
    Hk = rng.choice([1, 2, 4, 8, 16])
    Hv = Hk * rng.choice([1, 2, 2, 3, 4])
    dk, dv = rng.choice([(128, 128), (128, 128), (64, 128), (64, 64), (128, 64)])
    seed = rng.randint(1, 1 << 20)
    if kind == "block":
        dk = dv = 128
        B = rng.randint(1, 8)
        return _attn("", kind, B, rng.randint(1, 16 // B), Hk, Hv, dk, dv, seed, hidden=128 * _log(rng, 4, 40),
                     group=rng.choice([32, 64, 128]))
    rows = rng.choice([1, rng.randint(2, 9), _log(rng, 10, 100), _log(rng, 100, 8192)])
    c = _attn("", kind, _log(rng, 1, 64), rows, Hk, Hv, dk, dv, seed, fresh=rng.random() < 0.4,
              rule=rng.choice(["delta", "delta", "sum"]), gate=rng.random() < 0.5)
    while _cost(c) > most or c["B"] * c["rows"] > 16384:
        if c["B"] > 2:
            c["B"] = c["B"] * 3 // 4
        else:
            c["rows"] = c["rows"] * 3 // 4
    return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ---------------------------------------------------------------------------- inputs
def _gen(seed, what):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + what * 7919) & 0x7fffffffffff)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _uniform(g, lo, hi, *shape):
    return lo + (hi - lo) * torch.rand(*shape, generator=g, device=DEV, dtype=torch.float32)


def _rows(case):
    """New rows of every conversation: the first has ``rows``, those of a prompt call are ragged."""
    rng, r = random.Random(case["ragged"]), case["rows"]
    return [r if b == 0 or r <= 16 else rng.randint(max(1, r // 4), r) for b in range(case["B"])]


def _channels(case):
    return 2 * case["Hk"] * case["dk"] + case["Hv"] * case["dv"]


def _weight4(g, K, N, group, mins, scales):
    """A 4-bit weight whose values have a spread of about 1 / sqrt(K)."""
    codes = torch.randint(-(1 << 31), (1 << 31), (N, K // 8), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    to = torch.float16 if scales == "f16" else torch.float32
    scale = (_uniform(g, 0.5, 1.5, N, K // group) / (4.6 * math.sqrt(K))).to(to)
    return {"codes": codes, "scales": scale, "mins": (-_uniform(g, 6, 9, N, K // group) * scale.float()).to(to) if mins else None,
            "group": group}


def _layer(case, g):
    """A layer's parameters: convolution taps, decay rates and time-step offsets as such layers start from."""
    C, Hv = _channels(case), case["Hv"]
    dt = torch.exp(_uniform(g, math.log(1e-3), math.log(1e-1), Hv))
    return {"taps": _normal(g, C, TAPS) * 0.5, "a_log": torch.log(_uniform(g, 1, 16, Hv)),
            "dt_bias": dt + torch.log(-torch.expm1(-dt)), "norm": 1 + 0.1 * _normal(g, case["dv"])}


def prepare(case, seed):
    g = _gen(seed, 1)
    if case["op"] == "proj":
        M, K, N = case["M"], case["K"], case["N0"] + case["N1"] + case["N2"]
        s = {"case": case, "x": _normal(g, M, K), "w": _weight4(g, K, N, case["group"], case["mins"], case["scales"]),
             "resid": _normal(g, M, N) if case["resid"] else None}
        if own:
            s["handle"] = _handle(s["w"], K, case["N0"], case["N1"], case["N2"])
        return s
    rows, B, Hk, Hv, dk, dv = _rows(case), case["B"], case["Hk"], case["Hv"], case["dk"], case["dv"]
    T, C = sum(rows), _channels(case)
    slots = list(range(B + 1))  # one slot that no conversation of this batch holds
    random.Random(case["ragged"] + 1).shuffle(slots)
    slots = slots[:B]
    s = {"case": case, "rows": rows, "slots": slots, **_layer(case, g)}
    # what earlier calls left, stale values in the slots of new conversations included
    s["state"] = 0.1 * _normal(g, 1, B + 1, Hv, dv, dk)
    s["conv"] = _normal(g, 1, B + 1, TAPS - 1, C)
    silu = torch.nn.functional.silu
    if case["op"] == "block":
        h = case["hidden"]
        s["x"], s["h"] = _normal(g, T, h), _normal(g, T, h)
        s["w_in"] = _weight4(g, h, C + Hv * dv + 2 * Hv, case["group"], False, "f16")
        s["w_out"] = _weight4(g, Hv * dv, h, case["group"], False, "f16")
    elif case["op"] == "prologue":
        s["qkv"], s["a"], s["b"] = _normal(g, T, C), _normal(g, T, Hv), _normal(g, T, Hv)
    else:  # what a prologue gives
        s["q"], s["k"] = (_unit(silu(_normal(g, T, Hk, dk))) for _ in range(2))
        s["v"], s["z"] = silu(_normal(g, T, Hv, dv)), _normal(g, T, Hv, dv)
        s["g"] = -torch.exp(s["a_log"]) * torch.nn.functional.softplus(s["dt_bias"] + _normal(g, T, Hv))
        s["beta"] = torch.sigmoid(_normal(g, T, Hv)) if case["rule"] == "delta" else None
        if case["rule"] == "sum":
            s["g"] = -0.1 * torch.exp(s["a_log"]) / 16  # a constant for each head
    # the batch as device indices (the plain form's, and a user's own bookkeeping)
    first = np.concatenate([[0], np.cumsum(rows)[:-1]])
    seq = np.repeat(np.arange(B), rows)
    place = np.arange(T) - first[seq]
    back = place[:, None] - (TAPS - 1) + np.arange(TAPS)  # the rows each tap reads; below 0: kept inputs
    taps = np.where(back < 0, (TAPS - 1) * seq[:, None] + back + TAPS - 1, (TAPS - 1) * B + first[seq][:, None] + back)
    last = np.asarray(rows)[:, None] - (TAPS - 1) + np.arange(TAPS - 1)
    keep = np.where(last < 0, (TAPS - 1) * np.arange(B)[:, None] + last + TAPS - 1, (TAPS - 1) * B + first[:, None] + last)
    n = min(CHUNK, max(rows))
    padded = np.full((B, -(-max(rows) // n) * n), T, np.int64)  # T: a row of zeros
    padded[seq, place] = np.arange(T)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    s.update(seq=dev(seq), place=dev(place), tap_rows=dev(taps), keep_rows=dev(keep), padded=dev(padded), slots_dev=dev(np.asarray(slots)))
    if own:
        from bitgpu_amd import engine as E
        s["cache"] = E.LinearStateCache(1, Hk, Hv, dk, dv, n_slots=B + 1, conv_width=TAPS, state=s["state"], conv=s["conv"])
        s["batch"] = E.LinearBatch(s["cache"], max_seqs=B, max_tokens=T)
        s["batch"].set(rows, slots, sources=[-1] * B if case["fresh"] else None)
        if case["op"] == "block":
            s["in"] = _handle(s["w_in"], case["hidden"], C, Hv * dv, 2 * Hv)
            s["out"] = _handle(s["w_out"], Hv * dv, case["hidden"], 0, 0)
    return s


def _unit(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)


def _handle(w, K, N0, N1, N2):
    from bitgpu_amd import engine as E
    return E.FourBitWeight(w["codes"], w["scales"], K, N0, N1, N2, group=w["group"], mins=w["mins"])


# ---------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    return {"prologue": _run_prologue, "attention": _run_attention, "proj": _run_proj, "block": _run_block}[case["op"]](s)


def _run_prologue(s):
    if own:
        from bitgpu_amd import engine as E
        q, k, v, g, beta = E.linear_prologue(s["cache"], 0, s["batch"], s["qkv"], s["taps"], s["a"], s["b"], s["a_log"],
                                             s["dt_bias"])
    else:
        q, k, v, g, beta = _prologue(s, s["qkv"], s["a"], s["b"])
    return {"q": q, "k": k, "v": v, "g": g, "beta": beta, "conv": s["conv"]}


def _run_attention(s):
    gate = s["case"]["gate"]
    if own:
        from bitgpu_amd import engine as E
        o = E.linear_attention(s["cache"], 0, s["batch"], s["q"], s["k"], s["v"], s["g"], s["beta"], gate=s["z"] if gate else None,
                               norm=s["norm"] if gate else None, eps=EPS)
    else:
        o = _attention(s, s["q"], s["k"], s["v"], s["g"], s["beta"])
        o = _gated_norm(s, o, s["z"]) if gate else o
    return {"out": o, "state": s["state"]}


def _run_proj(s):
    case, x = s["case"], s["x"]
    if own:
        from bitgpu_amd import engine as E
        if case["resid"]:
            return E.resid_mm(s["handle"], x, s["resid"])
        outs = [x.new_empty(case["M"], n) for n in (case["N0"], case["N1"], case["N2"]) if n]
        E.fused_mm(s["handle"], x, outs)
        return outs
    y = _times(x, s["w"])
    if case["resid"]:
        return y + s["resid"]
    return [t.contiguous() for t in y.split([n for n in (case["N0"], case["N1"], case["N2"]) if n], 1)]


def _run_block(s):
    case = s["case"]
    if own:
        from bitgpu_amd import engine as E
        out = E.linear_block(s["cache"], 0, s["batch"], s["x"], s["h"], s["in"], s["out"], s["taps"], s["a_log"], s["dt_bias"],
                             s["norm"], EPS)
    else:
        C, Hv, dv = _channels(case), case["Hv"], case["dv"]
        qkv, z, b, a = _times(s["x"], s["w_in"]).split([C, Hv * dv, Hv, Hv], 1)
        o = _gated_norm(s, _attention(s, *_prologue(s, qkv, a, b)), z.reshape(-1, Hv, dv))
        out = _times(o.reshape(-1, Hv * dv), s["w_out"]) + s["h"]
    return {"out": out, "state": s["state"], "conv": s["conv"]}


def _prologue(s, qkv, a, b):
    case = s["case"]
    Hk, Hv, dk, dv = case["Hk"], case["Hv"], case["dk"], case["dv"]
    kept = s["conv"][0, s["slots_dev"]]
    if case["fresh"]:
        kept = torch.zeros_like(kept)
    inputs = torch.cat([kept.flatten(0, 1), qkv])
    y = (inputs[s["tap_rows"]] * s["taps"].T).sum(1)
    s["conv"][0, s["slots_dev"]] = inputs[s["keep_rows"]]
    y = y / (1 + torch.exp(-y))
    q, k, v = y.split([Hk * dk, Hk * dk, Hv * dv], 1)
    t = a + s["dt_bias"]
    softplus = t.clamp_min(0) + torch.log1p(torch.exp(-t.abs()))
    return (_unit(q.reshape(-1, Hk, dk)), _unit(k.reshape(-1, Hk, dk)), v.reshape(-1, Hv, dv).contiguous(),
            -torch.exp(s["a_log"]) * softplus, 1 / (1 + torch.exp(-b)))


def _attention(s, q, k, v, g, beta):
    """The recurrence a chunk of rows at a time. Within a chunk the rows' corrections depend on each other
    through I + A, A strictly lower triangular, whose inverse is the product of I + (-A)^(2^i); decays are sums
    over long spans and that product cancels, so both are taken in 64 bits."""
    case = s["case"]
    Hv, rep, dv = case["Hv"], case["Hv"] // case["Hk"], case["dv"]
    B, L = s["padded"].shape
    n = min(CHUNK, L)

    def chunked(x, heads):  # [T, heads, ...] -> [chunks, B, heads, n, ...], zeros behind each conversation's rows
        x = torch.cat([x, x.new_zeros(1, *x.shape[1:])])[s["padded"]].unflatten(1, (-1, n)).transpose(0, 1).transpose(2, 3)
        return x.repeat_interleave(heads, 2) if heads > 1 else x

    q, k, v = chunked(q, rep), chunked(k, rep), chunked(v, 1)
    live = chunked(torch.ones_like(s["place"], dtype=torch.float64)[:, None], 1)  # [chunks, B, 1, n]
    g = chunked(g.double(), 1) if g.dim() == 2 else g.double()[:, None] * live
    sums = g.cumsum(-1)  # [chunks, B, Hv, n]
    row = torch.arange(n, device=DEV)
    fade = (sums[..., :, None] - sums[..., None, :]).masked_fill(row[:, None] < row, -math.inf).exp()
    from_start, to_end = sums.exp().float()[..., None], (sums[..., -1:] - sums).exp().float()[..., None]
    whole = sums[..., -1, None, None].exp().float()
    scores = torch.matmul(q, k.transpose(-1, -2)) * fade.float()
    if beta is not None:
        beta = chunked(beta, 1)[..., None]
        power = -(beta * torch.matmul(k, k.transpose(-1, -2))).double() * fade
        power = power.masked_fill(row[:, None] == row, 0)
        inverse = torch.eye(n, device=DEV, dtype=torch.float64) + power
        for _ in range(max(0, (n - 1).bit_length() - 1)):
            power = torch.matmul(power, power)
            inverse = inverse + torch.matmul(inverse, power)
        inverse = inverse.float()
    state = s["state"][0, s["slots_dev"]].transpose(-1, -2)  # [B, Hv, dk, dv]
    if case["fresh"]:
        state = torch.zeros_like(state)
    outs = []
    for c in range(L // n):  # the recurrence itself
        new = v[c]
        if beta is not None:
            new = torch.matmul(inverse[c], beta[c] * (new - from_start[c] * torch.matmul(k[c], state)))
        outs.append(from_start[c] * torch.matmul(q[c], state) + torch.matmul(scores[c], new))
        state = whole[c] * state + torch.matmul((to_end[c] * k[c]).transpose(-1, -2), new)
    s["state"][0, s["slots_dev"]] = state.transpose(-1, -2)
    out = torch.stack(outs, 1).transpose(2, 3).reshape(B, L, Hv, dv)
    return out[s["seq"], s["place"]] / math.sqrt(case["dk"])


def _gated_norm(s, o, z):
    return o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm"] * (z / (1 + torch.exp(-z)))


def _values4(w):
    """A 4-bit weight as the values it stands for, [N, K]."""
    to = torch.float32
    c = (w["codes"][..., None] >> torch.arange(0, 32, 4, device=DEV, dtype=torch.int32)) & 15
    c = c.flatten(1).to(to).unflatten(1, (-1, w["group"]))
    scale = w["scales"].to(to)[..., None]
    y = c * scale + w["mins"].to(to)[..., None] if w["mins"] is not None else (c - 8) * scale
    return y.flatten(1)


def _times(x, w):
    return torch.matmul(x, _values4(w).T)


# ---------------------------------------------------------------------------- work and exact results
def work(case):
    if case["op"] == "proj":
        return _proj_work(case["M"], case["K"], case["N0"] + case["N1"] + case["N2"], case["group"],
                          (2 if case["scales"] == "f16" else 4) * (2 if case["mins"] else 1), case["resid"])
    rows, B, Hk, Hv, dk, dv = _rows(case), case["B"], case["Hk"], case["Hv"], case["dk"], case["dv"]
    T, C = sum(rows), _channels(case)
    states = 1 if case["fresh"] else 2  # written, and read where there is one
    prologue = {"bytes": 4 * (2 * T * C + 4 * T * Hv + states * B * (TAPS - 1) * C + TAPS * C), "flops": T * C * (2 * TAPS + 6)}
    attention = {"bytes": 4 * (T * C + T * Hv * (1 if case["rule"] == "sum" else 2) + T * Hv * dv * (2 if case["gate"] else 1)
                               + states * B * Hv * dk * dv),
                 "flops": T * Hv * dk * dv * (6 if case["rule"] == "delta" else 4)}
    if case["op"] == "prologue":
        return prologue
    if case["op"] == "attention":
        return attention
    h = case["hidden"]
    two = [_proj_work(T, h, C + Hv * dv + 2 * Hv, case["group"], 2, False), _proj_work(T, Hv * dv, h, case["group"], 2, True)]
    # between the operators: nothing that has to leave the chip but what the layer reads and writes
    return {"bytes": two[0]["bytes"] + two[1]["bytes"] - 4 * T * (C + 2 * Hv * dv + 2 * Hv)
            + 4 * (states * B * (Hv * dk * dv + (TAPS - 1) * C) + TAPS * C),
            "flops": two[0]["flops"] + two[1]["flops"] + prologue["flops"] + attention["flops"]}


def _proj_work(M, K, N, group, per_group, resid):
    return {"bytes": N * K / 2 + N * K / group * per_group + 4 * M * (K + N * (2 if resid else 1)), "flops": 2 * M * N * K}


def exact(case, seed):
    """The definitions in float64: one row after the other of all conversations."""
    s = prepare(case, seed)
    if case["op"] == "proj":
        y = _exact_times(s["x"].double(), s["w"])
        if case["resid"]:
            return y + s["resid"]
        return list(y.split([n for n in (case["N0"], case["N1"], case["N2"]) if n], 1))
    if case["op"] == "prologue":
        return _exact_prologue(s, s["qkv"].double(), s["a"].double(), s["b"].double())
    Hv, dv, C = case["Hv"], case["dv"], _channels(case)
    if case["op"] == "attention":
        got = {n: s[n].double() for n in ("q", "k", "v", "g")}
        o, state = _exact_attention(s, **got, beta=None if s["beta"] is None else s["beta"].double())
        return {"out": _exact_norm(s, o, s["z"].double()) if case["gate"] else o, "state": state}
    y = _exact_times(s["x"].double(), s["w_in"])
    z = y[:, C:C + Hv * dv].reshape(-1, Hv, dv)
    b, a = y[:, C + Hv * dv:C + Hv * dv + Hv], y[:, C + Hv * dv + Hv:]
    p = _exact_prologue(s, y[:, :C], a, b)
    o, state = _exact_attention(s, p["q"], p["k"], p["v"], p["g"], p["beta"])
    o = _exact_norm(s, o, z).reshape(-1, Hv * dv)
    return {"out": _exact_times(o, s["w_out"]) + s["h"], "state": state, "conv": p["conv"]}


def _exact_prologue(s, qkv, a, b):
    case = s["case"]
    Hk, Hv, dk, dv = case["Hk"], case["Hv"], case["dk"], case["dv"]
    conv, ys, at = s["conv"].double(), [], 0
    for r, slot in zip(s["rows"], s["slots"]):
        kept = conv[0, slot] * (0 if case["fresh"] else 1)
        x = torch.cat([kept, qkv[at:at + r]])
        ys.append(sum(x[j:j + r] * s["taps"][:, j].double() for j in range(TAPS)))
        conv[0, slot] = x[-(TAPS - 1):]
        at += r
    y = torch.cat(ys)
    y = y * torch.sigmoid(y)
    heads = y[:, :2 * Hk * dk].reshape(-1, 2 * Hk, dk)
    heads = heads / (heads.square().sum(-1, keepdim=True) + EPS).sqrt()
    t = a + s["dt_bias"].double()
    return {"q": heads[:, :Hk], "k": heads[:, Hk:], "v": y[:, 2 * Hk * dk:].reshape(-1, Hv, dv),
            "g": -torch.exp(s["a_log"].double()) * torch.logaddexp(t, torch.zeros_like(t)), "beta": torch.sigmoid(b),
            "conv": conv}


def _exact_attention(s, q, k, v, g, beta):
    case = s["case"]
    Hv, rep, T = case["Hv"], case["Hv"] // case["Hk"], v.shape[0]
    rows = np.asarray(s["rows"])
    first = np.concatenate([[0], np.cumsum(rows)[:-1]])
    state = s["state"].double()
    S = state[0, s["slots_dev"]] * (0 if case["fresh"] else 1)  # [B, Hv, dv, dk]
    fade = (g if g.dim() == 2 else g.expand(T, Hv)).exp()
    out = torch.empty_like(v)
    order = np.argsort(-rows, kind="stable")  # conversations by length, so that those with a row i come first
    S = S[torch.from_numpy(order).to(DEV)]
    starts = torch.from_numpy(first[order]).to(DEV)
    for i in range(int(rows.max())):
        m = int((rows > i).sum())
        at = starts[:m] + i
        kk = k[at].repeat_interleave(rep, 1)[..., None]
        part = S[:m] * fade[at][..., None, None]
        add = v[at]
        if beta is not None:
            add = beta[at][..., None] * (add - torch.matmul(part, kk)[..., 0])
        part = part + add[..., None] * kk.transpose(-1, -2)
        S[:m] = part
        out[at] = torch.matmul(part, q[at].repeat_interleave(rep, 1)[..., None])[..., 0]
    state[0, s["slots_dev"][torch.from_numpy(order).to(DEV)]] = S
    return out / math.sqrt(case["dk"]), state


def _exact_norm(s, o, z):
    return o * (o.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["norm"].double() * z * torch.sigmoid(z)


def _exact_times(x, w):
    N, words = w["codes"].shape
    c = torch.stack([torch.bitwise_and(torch.bitwise_right_shift(w["codes"], 4 * i), 15) for i in range(8)], -1)
    c = c.view(N, -1, w["group"]).double()
    m = -8 * w["scales"].double() if w["mins"] is None else w["mins"].double()
    W = (c * w["scales"].double()[..., None] + m[..., None]).view(N, 8 * words)
    return (W @ x.T).T
