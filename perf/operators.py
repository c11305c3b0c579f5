"""Cases and plain forms of the sequence operators: layer_norm, gru_scan and gated_mlp (motif_amd.ops), forward and training steps.

layer_norm   y = (x - mean) / sqrt(var + eps) * w + b over the last axis
gru_scan     h_t = (1 - z_t) h_{t-1} + z_t q_t, channel by channel along a sequence: gru_update over a whole sequence whose gates do not
             read the state.  [B, T, D], or [rows, D] with sequences packed one behind the other (cu_seqlens)
gated_mlp    h = act(x Wg^T + bg) * (x Wu^T + bu)
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5


def listed():
    return [
        # one decoding step's rows: a call that is all latency
        {"name": "layer_norm step", "op": "layer_norm", "train": False, "dtype": "bf16", "rows": 16, "d": 1024},
        # every pixel of a 180 x 320 feature map with the framework's 64 channels
        {"name": "layer_norm pixels", "op": "layer_norm", "train": True, "dtype": "fp32", "rows": 57600, "d": 64},
        # a training batch of tokens
        {"name": "layer_norm tokens", "op": "layer_norm", "train": True, "dtype": "bf16", "rows": 16384, "d": 4096},
        # rows of an odd length, none but the first aligned
        {"name": "layer_norm odd", "op": "layer_norm", "train": True, "dtype": "fp16", "rows": 4099, "d": 1001},
        # one token for each of 64 streams, their states carried along
        {"name": "gru_scan step", "op": "gru_scan", "train": False, "dtype": "bf16", "b": 64, "t": 1, "d": 2048, "packed": 0},
        # the seven frames of a clip, each pixel and channel of a 64 x 180 x 320 feature map a sequence of its own
        {"name": "gru_scan clip", "op": "gru_scan", "train": False, "dtype": "fp32", "b": 1, "t": 7, "d": 64 * 180 * 320, "packed": 0},
        # one long sequence in training
        {"name": "gru_scan long", "op": "gru_scan", "train": True, "dtype": "bf16", "b": 1, "t": 65536, "d": 1024, "packed": 0},
        # sequences of very different lengths, some empty, packed; an odd width
        {"name": "gru_scan packed", "op": "gru_scan", "train": True, "dtype": "fp16", "b": 1, "t": 20011, "d": 771, "packed": 37},
        # one token
        {"name": "gated_mlp step", "op": "gated_mlp", "train": False, "dtype": "bf16", "m": 1, "k": 2048, "f": 5632, "act": "silu", "bias": False},
        # the pixels of a 180 x 320 feature map through 64 -> 256 channels, in the framework's own type
        {"name": "gated_mlp pixels", "op": "gated_mlp", "train": True, "dtype": "fp32", "m": 57600, "k": 64, "f": 256, "act": "gelu", "bias": True},
        # a training batch of tokens
        {"name": "gated_mlp tokens", "op": "gated_mlp", "train": True, "dtype": "bf16", "m": 8192, "k": 2048, "f": 5632, "act": "silu", "bias": False},
        # sizes that no tile divides
        {"name": "gated_mlp ragged", "op": "gated_mlp", "train": True, "dtype": "fp16", "m": 1337, "k": 1000, "f": 2730, "act": "sigmoid", "bias": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size spread over its logarithm: every second one a multiple of 64, the others as they fall."""
    n = _log(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 and n >= 64 else n


def draw(rng):
    op = rng.choice(["layer_norm", "gru_scan", "gated_mlp"])
    case = {"op": op, "train": rng.random() < 0.6, "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    if op == "layer_norm":
        d = _size(rng, 32, 16384)
        return dict(case, rows=_log(rng, 1, min(1 << 19, (1 << 26) // d)), d=d)
    if op == "gru_scan":
        packed = rng.choice([0, 0, _log(rng, 2, 200)])
        d = _size(rng, 16, 1 << 20)
        t = _log(rng, 1, min(65536, max(1, (1 << 26) // d)))
        b = 1 if packed else _log(rng, 1, max(1, min(512, (1 << 26) // (d * t))))
        return dict(case, b=b, t=max(t, 2 * packed) if packed and d * 2 * packed <= 1 << 26 else t, d=d, packed=packed)
    k, f = _size(rng, 48, 4096), _size(rng, 48, 8192)
    most = 8192 * 2048 * 5632 // (k * f) // (3 if case["dtype"] == "fp32" else 1)
    return dict(case, m=_log(rng, 1, max(1, min(65536, most))), k=k, f=f, act=rng.choice(["silu", "gelu", "sigmoid"]), bias=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------------------------ inputs
def _bounds(case, seed):
    """Bounds of the packed sequences: a few empty, one of a single row, the others ragged; a few rows behind the last."""
    n, t = case["packed"], case["t"]
    g = torch.Generator().manual_seed(seed)
    share = -torch.log(torch.rand(n, generator=g, dtype=torch.float64).clamp_min(1e-9))
    share = share * (torch.rand(n, generator=g) > 0.1)
    share[0] += 1e-3
    used = max(1, t - t // 50)
    ends = (share.cumsum(0) / share.sum() * used).round().to(torch.int32)
    return torch.cat([torch.zeros(1, dtype=torch.int32), ends]).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["train"]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    s = {"op": case["op"], "train": train}
    if case["op"] == "layer_norm":
        d = case["d"]
        s["x"] = normal(case["rows"], d, scale=1.5, shift=0.3)
        s["w"], s["b"] = normal(d, scale=0.2, shift=1.0), normal(d, scale=0.2)
        s["dy"] = normal(case["rows"], d)
        s["leaves"] = ("x", "w", "b")
    elif case["op"] == "gru_scan":
        n = case["packed"]
        shape = (case["t"], case["d"]) if n else (case["b"], case["t"], case["d"])
        s["cu"] = _bounds(case, seed) if n else None
        s["z"] = torch.sigmoid(normal(*shape, scale=1.5, shift=-2.0, dtype=torch.float32)).to(dt)  # gates: mostly far from 1, a long memory
        s["q"] = torch.tanh(normal(*shape, dtype=torch.float32)).to(dt)
        s["h0"] = normal(n or case["b"], case["d"], scale=0.5, dtype=torch.float32)
        s["dh"], s["dlast"] = (normal(*shape), normal(n or case["b"], case["d"], dtype=torch.float32)) if train else (None, None)
        s["leaves"] = ("z", "q", "h0")
    else:
        m, k, f = case["m"], case["k"], case["f"]
        s["act"] = case["act"]
        s["x"] = normal(m, k)
        s["wg"], s["wu"] = normal(f, k, scale=k ** -0.5), normal(f, k, scale=k ** -0.5)
        s["bg"], s["bu"] = (normal(f, scale=0.1), normal(f, scale=0.1)) if case["bias"] else (None, None)
        s["dh"] = normal(m, f) if train else None
        s["leaves"] = ("x", "wg", "wu") + (("bg", "bu") if case["bias"] else ())
    if train:
        for name in s["leaves"]:
            s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _layer_norm(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    r = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = c * r
    out = [(n * w + b).to(s["x"].dtype)]
    if s["train"]:
        dy = s["dy"].float()
        dn = dy * w
        dx = r * (dn - dn.mean(-1, keepdim=True) - n * (dn * n).mean(-1, keepdim=True))
        out += [dx.to(s["x"].dtype), (dy * n).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)]
    return out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1, by doubling: after the step of n, a row holds the product and the sum of its last 2 n rows."""
    n = 1
    while n < a.shape[1]:
        b = torch.cat([b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]], 1)
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return b


def _gru_scan(s):
    dt, cu, h0 = s["q"].dtype, s["cu"], s["h0"]
    z, q = s["z"].float(), s["q"].float()
    if cu is not None:
        z, q = z[None], q[None]
    t = z.shape[1]
    row = torch.arange(t, device=z.device)
    if cu is None:
        first, owner, inside = (row == 0)[None, :], None, torch.ones(1, t, dtype=torch.bool, device=z.device)
        last = first.flip(1)
        init = torch.zeros_like(z)
        init[:, 0] = h0
    else:
        owner = (torch.searchsorted(cu, row.to(torch.int32), right=True) - 1).clamp(0, len(cu) - 2)
        inside = (row < cu[-1])[None, :]
        first, last = (row == cu[owner])[None, :] & inside, (row + 1 == cu[owner + 1])[None, :] & inside
        init = h0[owner][None] * first[..., None]
    z, q = (torch.where(inside[..., None], x, 0) for x in (z, q))  # rows behind the last sequence, whatever they hold
    a, u = 1 - z, z * q
    h = _scan(a * (~first)[..., None], u + a * init) * inside[..., None]
    if cu is None:
        end = h[:, -1]
    else:
        ends = cu[1:].long()
        empty = cu[1:] == cu[:-1]
        end = torch.where(empty[:, None], h0, h[0][(ends - 1).clamp_min(0)])
    out = [(h[0] if cu is not None else h).to(dt), end]
    if s["train"]:
        dh, dlast = s["dh"].float(), s["dlast"]
        if cu is None:
            dh = dh.clone()
            dh[:, -1] += dlast
        else:
            dh = torch.where(inside[..., None], dh[None] + dlast[owner][None] * last[..., None], 0)
        follow = torch.cat([a[:, 1:] * (~first[:, 1:])[..., None], torch.zeros_like(a[:, :1])], 1)
        g = _scan(follow.flip(1), dh.flip(1)).flip(1)
        before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1) * (~first)[..., None] + init
        dz, dq = g * (q - before), g * z
        da = g * a
        if cu is None:
            dh0 = da[:, 0]
        else:
            dz, dq = dz[0], dq[0]
            dh0 = torch.where(empty[:, None], dlast, da[0][cu[:-1].long().clamp_max(t - 1)])
        out += [dz.to(dt), dq.to(dt), dh0]
    return out


def _gate(g, act):
    """act(g) and its derivative."""
    sg = torch.sigmoid(g)
    if act == "sigmoid":
        return sg, sg * (1 - sg)
    if act == "silu":
        return g * sg, sg * (1 + g * (1 - sg))
    phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))


def _gated_mlp(s):
    dt = s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    if s["bg"] is not None:
        g, u = g + s["bg"].float(), u + s["bu"].float()
    v, dv = _gate(g, s["act"])
    out = [(v * u).to(dt)]
    if s["train"]:
        dh = s["dh"].float()
        dg, du = dh * u * dv, dh * v
        out += [(dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)]
        if s["bg"] is not None:
            out += [dg.sum(0).to(dt), du.sum(0).to(dt)]
    return out


def run(state):
    s = state
    if own:
        from motif_amd import ops
        if s["op"] == "layer_norm":
            y, dy = [ops.layer_norm(s["x"], s["w"], s["b"], eps=EPS)], [s["dy"]]
        elif s["op"] == "gru_scan":
            y, dy = list(ops.gru_scan(s["z"], s["q"], s["h0"], cu_seqlens=s["cu"])), [s["dh"], s["dlast"]]
        else:
            y, dy = [ops.gated_mlp(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], act=s["act"])], [s["dh"]]
        return y + list(torch.autograd.grad(y, [s[n] for n in s["leaves"]], dy)) if s["train"] else y
    with torch.no_grad():
        return {"layer_norm": _layer_norm, "gru_scan": _gru_scan, "gated_mlp": _gated_mlp}[s["op"]](s)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    train = case["train"]
    if case["op"] == "layer_norm":
        n, d = case["rows"] * case["d"], case["d"]
        # forward: x in, y out; backward: dy in, dx and the parameters' gradients out
        return {"bytes": e * ((4 if train else 2) * n + (4 if train else 2) * d), "flops": (20 if train else 8) * n}
    if case["op"] == "gru_scan":
        n = case["b"] * case["t"] * case["d"]
        states = (case["packed"] or case["b"]) * case["d"]
        # forward: z, q, h0 in, h and the last states out; backward: the outputs' gradients in, three gradients out
        return {"bytes": e * (6 if train else 3) * n + 4 * (4 if train else 2) * states, "flops": (12 if train else 4) * n}
    m, k, f = case["m"], case["k"], case["f"]
    weights = 2 * f * k + (2 * f if case["bias"] else 0)
    return {"bytes": e * ((2 if train else 1) * (m * k + weights) + (2 if train else 1) * m * f), "flops": (12 if train else 4) * m * k * f}


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        d = {n: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for n, v in s.items()}
        if case["op"] == "layer_norm":
            var, mean = torch.var_mean(d["x"], -1, correction=0, keepdim=True)
            std = torch.sqrt(var + EPS)
            hat = (d["x"] - mean) / std
            res = [hat * d["w"] + d["b"]]
            if case["train"]:
                up = d["dy"] * d["w"]
                along = (up * hat).mean(-1, keepdim=True)
                res += [(up - up.mean(-1, keepdim=True) - hat * along) / std, torch.einsum("rd,rd->d", d["dy"], hat), d["dy"].sum(0)]
            return res
        if case["op"] == "gated_mlp":
            pre = [torch.nn.functional.linear(d["x"], d[w], d[b]) for w, b in (("wg", "bg"), ("wu", "bu"))]
            pre = [p.requires_grad_() for p in pre]
            with torch.enable_grad():
                val = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid}[case["act"]](pre[0]) * pre[1]
                got = torch.autograd.grad(val, pre, d["dh"]) if case["train"] else []
            res = [val]
            if case["train"]:
                res += [torch.matmul(got[0], d["wg"]) + torch.matmul(got[1], d["wu"])] + [torch.matmul(p.t(), d["x"]) for p in got]
                res += [p.sum(0) for p in got] if case["bias"] else []
            return res
        return _exact_scan(case, s, d)


def _exact_scan(case, s, d):
    """Row by row, as the recurrence is written."""
    z, q, dh = d["z"], d["q"], d["dh"]
    if case["packed"]:
        bounds = s["cu"].tolist()
        spans = [(i, bounds[i], bounds[i + 1]) for i in range(case["packed"])]
        rows = lambda x, lo, hi: x[lo:hi].unsqueeze(0)  # noqa: E731
    else:
        spans = [(slice(None), 0, case["t"])]
        rows = lambda x, lo, hi: x[:, lo:hi]  # noqa: E731
    h, last = torch.zeros_like(q), d["h0"].clone()
    dz, dq, dh0 = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(last)
    for i, lo, hi in spans:
        zi, qi, hi_ = rows(z, lo, hi), rows(q, lo, hi), rows(h, lo, hi)
        begin = d["h0"][i].reshape(-1, case["d"])
        state = begin
        for t in range(hi - lo):
            state = torch.lerp(state, qi[:, t], zi[:, t])
            hi_[:, t] = state
        last[i] = state.reshape(last[i].shape)
        if case["train"]:
            back = d["dlast"][i].reshape(-1, case["d"])
            di, dzi, dqi = rows(dh, lo, hi), rows(dz, lo, hi), rows(dq, lo, hi)
            for t in range(hi - lo - 1, -1, -1):
                back = back + di[:, t]
                dzi[:, t] = back * (qi[:, t] - (hi_[:, t - 1] if t else begin))
                dqi[:, t] = back * zi[:, t]
                back = back - back * zi[:, t]
            dh0[i] = back.reshape(dh0[i].shape)
    return [h, last] + ([dz, dq, dh0] if case["train"] else [])
