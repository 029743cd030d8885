"""Measured cases of the selective-scan serving operators.

Four operators carry a selective state space model through serving: the short
causal convolution and the selective scan over prompts (CausalConv1dFn,
SelectiveScanVarlenFn: packed or batched sequences that may continue cached
states) and over single tokens (CausalConv1dUpdateFn, SelectiveStateUpdateFn).
`listed()` and `draw()` give the cases, `prepare()` what a program holds before
the call, `run()` one pass (the plain torch form, or the library's kernels where
`own` is true), `exact()` the definition in 64 bits, `work()` the bytes and
operations a pass cannot do without.
"""

import importlib.util
import math
import pathlib
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_PKG_DIR = pathlib.Path(__file__).resolve().parents[1] / "xmetai-onnx-plugins_b200"
_PKG = "xmetai_onnx_plugins_b200"


def _package():
    """The library's Python package (its directory name has dashes)."""
    mod = sys.modules.get(_PKG)
    if mod is None:
        spec = importlib.util.spec_from_file_location(_PKG, _PKG_DIR / "__init__.py",
                                                      submodule_search_locations=[str(_PKG_DIR)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[_PKG] = mod
        spec.loader.exec_module(mod)
    return mod


# ------------------------------------------------------------------ cases


def listed():
    return [
        # A prefill step of a server: ragged prompts packed into one row, token-major as the projections
        # leave them, some continuing a cached state, all states in a pool of slots.
        dict(name="conv_prompts_packed", op="conv", dtype="bfloat16", layout="tokens", packed=True, units=24,
             tokens=16384, dim=4096, width=4, bias=True, silu=True, state="pool"),
        # The benchmark configuration's batch of 2048-token prompts, channel-major as SelectiveScanFn takes it.
        dict(name="conv_batch_channel_major", op="conv", dtype="bfloat16", layout="channels", packed=False, units=8,
             tokens=16384, dim=4096, width=4, bias=True, silu=True, state="none"),
        # A small model in float32 with an odd length, continuing given states (chunked prefill).
        dict(name="conv_small_odd", op="conv", dtype="float32", layout="channels", packed=False, units=2,
             tokens=514, dim=64, width=4, bias=True, silu=True, state="rows"),
        # One sequence decoding one token: latency.
        dict(name="conv_token_single", op="conv_token", dtype="bfloat16", batch=1, dim=4096, width=4, bias=True,
             silu=True, slots=0),
        # A full decode batch over a pool of slots.
        dict(name="conv_token_batch", op="conv_token", dtype="float16", batch=256, dim=4096, width=4, bias=True,
             silu=True, slots=320),
        # The packed prefill step's scan.
        dict(name="scan_prompts_packed", op="scan", dtype="bfloat16", packed=True, units=24, tokens=16384, dim=4096,
             dstate=16, groups=1, gate=True, state="pool"),
        # One long document: few channel rows, a long axis.
        dict(name="scan_long_document", op="scan", dtype="bfloat16", packed=False, units=1, tokens=32768, dim=2048,
             dstate=16, groups=1, gate=True, state="rows"),
        # The benchmark configuration's batch (8 x 2048 tokens, 4096 channels).
        dict(name="scan_batch", op="scan", dtype="bfloat16", packed=False, units=8, tokens=16384, dim=4096, dstate=16,
             groups=1, gate=True, state="none"),
        # A small model in float32, odd length, no gate, states given and returned.
        dict(name="scan_small_odd", op="scan", dtype="float32", packed=False, units=2, tokens=514, dim=64, dstate=16,
             groups=1, gate=False, state="rows"),
        # One sequence decoding one token: latency.
        dict(name="token_single", op="token", dtype="bfloat16", batch=1, dim=4096, dstate=16, groups=1, gate=True,
             slots=0),
        # A full decode batch over a pool of slots.
        dict(name="token_batch", op="token", dtype="bfloat16", batch=256, dim=4096, dstate=16, groups=1, gate=True,
             slots=320),
        # The largest decode batch, wider states in groups, float32 activations.
        dict(name="token_batch_wide", op="token", dtype="float32", batch=512, dim=2048, dstate=64, groups=2,
             gate=True, slots=0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _round_dim(rng, n):
    """Most models' widths are multiples of 64; some are not."""
    return max(64, n // 64 * 64) if rng.random() < 0.7 else n


def draw(rng):
    op = rng.choice(["conv", "conv_token", "scan", "token"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    size = 4 if dtype == "float32" else 2
    dim = _round_dim(rng, _log_int(rng, 48, 8192))
    if op == "conv":
        most = (1 << 26) * 2 // size // dim
        packed = rng.random() < 0.5
        tokens = _log_int(rng, 1, min(65536, most))
        units = _log_int(rng, 1, max(1, min(64, tokens)))
        if not packed:
            tokens = max(1, tokens // units) * units
        return dict(op=op, dtype=dtype, layout=rng.choice(["tokens", "channels"]), packed=packed, units=units,
                    tokens=tokens, dim=dim, width=rng.choice([2, 3, 4, 4]), bias=rng.random() < 0.7,
                    silu=rng.random() < 0.8, state=rng.choice(["none", "rows", "pool"]))
    if op == "conv_token":
        batch = _log_int(rng, 1, 1024)
        return dict(op=op, dtype=dtype, batch=batch, dim=dim, width=rng.choice([2, 3, 4, 4]),
                    bias=rng.random() < 0.7, silu=rng.random() < 0.8,
                    slots=rng.choice([0, batch + rng.randint(0, 64)]))
    dstate = rng.choice([8, 16, 16, 16, 32, 64, 128, rng.randint(1, 200)])
    groups = rng.choice([1, 1, 2, 4])
    dim = dim // groups * groups
    if op == "scan":
        most = (1 << 30) // (dim * max(16, dstate)) * 2 // size
        packed = rng.random() < 0.5
        tokens = _log_int(rng, 1, min(16384, most))
        units = _log_int(rng, 1, max(1, min(48, tokens)))
        if not packed:
            tokens = max(1, tokens // units) * units
        return dict(op=op, dtype=dtype, packed=packed, units=units, tokens=tokens, dim=dim, dstate=dstate,
                    groups=groups, gate=rng.random() < 0.7, state=rng.choice(["none", "rows", "pool"]))
    batch = _log_int(rng, 1, max(1, min(1024, (1 << 26) // (dim * dstate))))
    return dict(op=op, dtype=dtype, batch=batch, dim=dim, dstate=dstate, groups=groups, gate=rng.random() < 0.7,
                slots=rng.choice([0, batch + rng.randint(0, 64)]))


# ------------------------------------------------------------------ inputs


class _Maker:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) * 7919 + 17)

    def normal(self, shape, dtype=torch.float32, std=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(dtype)

    def uniform(self, shape, lo, hi, dtype=torch.float32):
        return (torch.rand(shape, generator=self.g, device="cuda") * (hi - lo) + lo).to(dtype)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _offsets(m, case):
    """Sequence boundaries: equal rows of a batch, or ragged packed lengths (log-normal, at least one token)."""
    units, tokens = case["units"], case["tokens"]
    if not case["packed"]:
        return [i * (tokens // units) for i in range(units + 1)]
    w = torch.exp(0.8 * m.normal((units,))).double().cpu()
    ends = torch.round(torch.cumsum(w, 0) / w.sum() * (tokens - units)).long().tolist()
    return [0] + [e + i + 1 for i, e in enumerate(ends)]


def _with_states(m, s, case, shape, dtype, std):
    """The recurrent states of the case: none, one row per sequence, or a pool addressed by slot numbers in
    which about half of the sequences begin anew."""
    s["state"] = s["slots"] = s["live"] = None
    units = case["units"]
    if case["state"] == "rows":
        s["state"] = m.normal((units, *shape), dtype, std)
    elif case["state"] == "pool":
        n = units + 16
        s["state"] = m.normal((n, *shape), dtype, std)
        s["slots"] = m.perm(n)[:units].to(torch.int32)
        s["live"] = (m.uniform((units,), 0, 1) < 0.5).to(torch.int32)


def _ssm_params(m, s, dim, dstate):
    # A[d, n] = -(n + 1); steps softplus(N(0, 1) + softplus^-1(U[0.001, 0.1])); D = 1 (the benchmark's values)
    s["A"] = -(torch.arange(dstate, device="cuda", dtype=torch.float32) + 1).repeat(dim, 1)
    s["D"] = torch.ones(dim, device="cuda")
    s["delta_bias"] = torch.log(torch.expm1(m.uniform((dim,), 0.001, 0.1)))


def prepare(case, seed):
    m, op, dt = _Maker(seed), case["op"], DTYPES[case["dtype"]]
    s = {"case": case}
    if op in ("conv", "conv_token"):
        dim, width = case["dim"], case["width"]
        s["weight"] = m.uniform((dim, width), -width ** -0.5, width ** -0.5)
        s["bias"] = m.uniform((dim,), -0.5, 0.5) if case["bias"] else None
        if op == "conv_token":
            n = case["slots"] or case["batch"]
            s["x"] = m.normal((case["batch"], dim), dt)
            s["state"] = m.normal((n, dim, width - 1), dt)
            s["slots"] = m.perm(n)[:case["batch"]].to(torch.int32) if case["slots"] else None
            return s
        cu = _offsets(m, case)
        rows, length = (1, case["tokens"]) if case["packed"] else (case["units"], case["tokens"] // case["units"])
        s["x"] = m.normal((rows, length, dim) if case["layout"] == "tokens" else (rows, dim, length), dt)
        _with_states(m, s, case, (dim, width - 1), dt, 1.0)
    else:
        dim, dstate, groups = case["dim"], case["dstate"], case["groups"]
        _ssm_params(m, s, dim, dstate)
        if op == "token":
            batch = case["batch"]
            n = case["slots"] or batch
            s["u"], s["delta"] = m.normal((batch, dim), dt), m.normal((batch, dim), dt)
            s["z"] = m.normal((batch, dim), dt) if case["gate"] else None
            s["B"], s["C"] = m.normal((batch, groups, dstate), dt), m.normal((batch, groups, dstate), dt)
            s["state"] = m.normal((n, dim, dstate), std=0.5)
            s["slots"] = m.perm(n)[:batch].to(torch.int32) if case["slots"] else None
            return s
        cu = _offsets(m, case)
        rows, length = (1, case["tokens"]) if case["packed"] else (case["units"], case["tokens"] // case["units"])
        s["u"], s["delta"] = m.normal((rows, length, dim), dt), m.normal((rows, length, dim), dt)
        s["z"] = m.normal((rows, length, dim), dt) if case["gate"] else None
        s["B"] = m.normal((rows, length, groups, dstate), dt)
        s["C"] = m.normal((rows, length, groups, dstate), dt)
        _with_states(m, s, case, (dim, dstate), torch.float32, 0.5)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    s["longest"] = max(b - a for a, b in zip(cu, cu[1:]))
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    op = s["case"]["op"]
    if own:
        return {"conv": _own_conv, "conv_token": _own_conv_token, "scan": _own_scan, "token": _own_token}[op](s)
    return {"conv": _plain_conv, "conv_token": _plain_conv_token, "scan": _plain_scan, "token": _plain_token}[op](s)


def _own_conv(s):
    c = s["case"]
    return _package().CausalConv1dFn(
        s["x"], s["weight"], s["bias"], s["state"], s["cu"] if c["packed"] else None, s["slots"], s["live"],
        silu=int(c["silu"]), channels_last=int(c["layout"] == "tokens"),
        output_final_state=int(c["state"] != "none"))


def _own_conv_token(s):
    return _package().CausalConv1dUpdateFn(s["x"], s["weight"], s["bias"], s["state"], s["slots"],
                                           silu=int(s["case"]["silu"]))


def _own_scan(s):
    c = s["case"]
    return _package().SelectiveScanVarlenFn(
        s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"], s["delta_bias"], s["state"],
        s["cu"] if c["packed"] else None, s["slots"], s["live"], delta_softplus=1,
        output_final_state=int(c["state"] != "none"))


def _own_token(s):
    return _package().SelectiveStateUpdateFn(s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"],
                                             s["delta_bias"], s["state"], s["slots"], delta_softplus=1)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20))))


def _start_rows(s, shape):
    """The states that the sequences start from, in float32 (zeros where there are none)."""
    units = s["case"]["units"]
    if s["state"] is None:
        return torch.zeros((units, *shape), device="cuda")
    rows = s["state"] if s["slots"] is None else s["state"][s["slots"].long()]
    rows = rows.float()
    if s["live"] is not None:
        rows = torch.where(s["live"].view(-1, 1, 1) != 0, rows, torch.zeros_like(rows))
    return rows


def _end_rows(s, out, rows):
    if s["state"] is None:
        return out
    if s["slots"] is None:
        return out, rows.to(s["state"].dtype)
    s["state"][s["slots"].long()] = rows.to(s["state"].dtype)
    return out, s["state"]


def _plain_conv(s):
    c = s["case"]
    dim, width, units = c["dim"], c["width"], c["units"]
    x = s["x"] if c["layout"] == "tokens" else s["x"].transpose(1, 2)
    shape = x.shape
    x = x.reshape(-1, dim).float()
    cu = s["cu"].long()
    start = _start_rows(s, (dim, width - 1))
    # one row of `width - 1` starting values before every sequence's tokens
    t = torch.arange(x.shape[0], device=x.device)
    seq = torch.bucketize(t, cu[1:], right=True)
    ext = torch.empty((x.shape[0] + units * (width - 1), dim), device=x.device)
    at = t + (seq + 1) * (width - 1)
    ext[at] = x
    head = cu[:-1].view(-1, 1) + torch.arange(units, device=x.device).view(-1, 1) * (width - 1) + torch.arange(
        width - 1, device=x.device)
    ext[head.reshape(-1)] = start.transpose(1, 2).reshape(-1, dim)
    y = torch.zeros_like(x) if s["bias"] is None else s["bias"].expand_as(x)
    for k in range(width):
        y = y + ext[at - (width - 1) + k] * s["weight"][:, k]
    if c["silu"]:
        y = _silu(y)
    y = y.to(s["x"].dtype).reshape(shape)
    y = y if c["layout"] == "tokens" else y.transpose(1, 2).contiguous()
    last = cu[1:].view(-1, 1) + torch.arange(1, units + 1, device=x.device).view(-1, 1) * (width - 1) + torch.arange(
        -(width - 1), 0, device=x.device)
    return _end_rows(s, y, ext[last.reshape(-1)].reshape(units, width - 1, dim).transpose(1, 2).contiguous())


def _plain_conv_token(s):
    c = s["case"]
    old = s["state"] if s["slots"] is None else s["state"][s["slots"].long()]
    window = torch.cat([old, s["x"].unsqueeze(-1)], -1)
    y = (window.float() * s["weight"]).sum(-1)
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["silu"]:
        y = _silu(y)
    if s["slots"] is None:
        s["state"].copy_(window[..., 1:])
    else:
        s["state"][s["slots"].long()] = window[..., 1:]
    return y.to(s["x"].dtype), s["state"]


def _plain_scan(s):
    c = s["case"]
    dim, dstate, groups, units = c["dim"], c["dstate"], c["groups"], c["units"]
    tokens, longest = c["tokens"], s["longest"]
    flat = lambda v: v.reshape(tokens, *v.shape[2:])  # noqa: E731
    u, delta, B, C = flat(s["u"]), flat(s["delta"]), flat(s["B"]), flat(s["C"])
    z = None if s["z"] is None else flat(s["z"])
    cu = s["cu"].long()
    h = _start_rows(s, (dim, dstate))
    out = torch.empty_like(u)
    step = max(1, min(longest, (1 << 26) // (units * dim * dstate)))
    per = dim // groups
    wide = lambda v: v.repeat_interleave(per, dim=2) if groups > 1 else v  # noqa: E731
    for t0 in range(0, longest, step):
        t = torch.arange(t0, min(t0 + step, longest), device=u.device).view(-1, 1)
        at = cu[:-1].view(1, -1) + t
        inside = at < cu[1:].view(1, -1)
        at = torch.where(inside, at, torch.zeros_like(at))
        d = _softplus(delta[at].float() + s["delta_bias"])
        d = torch.where(inside.unsqueeze(-1), d, torch.zeros_like(d))
        uu = u[at].float()
        a = torch.exp(d.unsqueeze(-1) * s["A"])
        b = (d * uu).unsqueeze(-1) * wide(B[at].float())
        for i in range(a.shape[0]):
            h = torch.addcmul(b[i], a[i], h, out=b[i])
        y = (b * wide(C[at].float())).sum(-1) + s["D"] * uu
        if z is not None:
            y = y * _silu(z[at].float())
        out[at[inside]] = y[inside].to(out.dtype)
        h = h.clone()
    return _end_rows(s, out.reshape(s["u"].shape), h)


def _plain_token(s):
    c = s["case"]
    dim, groups = c["dim"], c["groups"]
    wide = lambda v: v.float().repeat_interleave(dim // groups, dim=1)  # noqa: E731
    old = s["state"] if s["slots"] is None else s["state"][s["slots"].long()]
    u = s["u"].float()
    d = _softplus(s["delta"].float() + s["delta_bias"])
    new = torch.exp(d.unsqueeze(-1) * s["A"]) * old + (d * u).unsqueeze(-1) * wide(s["B"])
    y = (new * wide(s["C"])).sum(-1) + s["D"] * u
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    if s["slots"] is None:
        s["state"].copy_(new)
    else:
        s["state"][s["slots"].long()] = new
    return y.to(s["u"].dtype), s["state"]


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "conv_token": _exact_conv_token, "scan": _exact_scan, "token": _exact_token}[
        case["op"]](s)


def _states64(s, end):
    if s["state"] is None:
        return None
    if s["slots"] is None:
        return end
    pool = s["state"].double()
    for i, slot in enumerate(s["slots"].tolist()):
        pool[slot] = end[i]
    return pool


def _exact_conv(s):
    c = s["case"]
    tail, bounds = c["width"] - 1, s["cu"].tolist()
    by_token = s["x"] if c["layout"] == "tokens" else s["x"].transpose(1, 2)
    x, w = by_token.reshape(-1, c["dim"]).double(), s["weight"].double()
    y, ends = torch.empty_like(x), []
    for i, (a, b) in enumerate(zip(bounds, bounds[1:])):
        start = torch.zeros((tail, c["dim"]), dtype=torch.float64, device=x.device)
        if s["state"] is not None and (s["live"] is None or int(s["live"][i])):
            start = s["state"][i if s["slots"] is None else int(s["slots"][i])].double().t()
        row = torch.cat([start, x[a:b]])
        # windows [tokens, dim, width] of the extended sequence
        v = (row.unfold(0, c["width"], 1) * w).sum(-1)
        if s["bias"] is not None:
            v += s["bias"].double()
        y[a:b] = v * torch.sigmoid(v) if c["silu"] else v
        ends.append(row[row.shape[0] - tail:].t())
    y = y.reshape(by_token.shape)
    y = y if c["layout"] == "tokens" else y.transpose(1, 2).contiguous()
    pool = _states64(s, torch.stack(ends))
    return y if pool is None else (y, pool)


def _exact_conv_token(s):
    y = torch.empty(s["x"].shape, dtype=torch.float64, device=s["x"].device)
    pool = s["state"].double()
    for b in range(s["x"].shape[0]):
        slot = b if s["slots"] is None else int(s["slots"][b])
        row = torch.cat([pool[slot], s["x"][b].double().unsqueeze(1)], 1)
        v = torch.einsum("dk,dk->d", row, s["weight"].double())
        if s["bias"] is not None:
            v = v + s["bias"].double()
        y[b] = v * torch.sigmoid(v) if s["case"]["silu"] else v
        pool[slot] = row[:, 1:]
    return y, pool


def _exact_scan(s):
    # h_t = a_t h_(t-1) + b_t over all packed tokens at once, by doubling: after the steps 1, 2, 4, ... the pair
    # (a_t, b_t) composes every step since the sequence's start, which carries the starting state in b and a = 0.
    c = s["case"]
    dim, dstate, groups, tokens = c["dim"], c["dstate"], c["groups"], c["tokens"]
    bounds = s["cu"].tolist()
    flat = lambda v: v.reshape(tokens, *v.shape[2:])  # noqa: E731
    y = torch.empty((tokens, dim), dtype=torch.float64, device="cuda")
    ends = torch.empty((c["units"], dim, dstate), dtype=torch.float64, device="cuda")
    first = torch.tensor(bounds[:-1], device="cuda")
    last = torch.tensor(bounds[1:], device="cuda") - 1
    per = dim // groups
    width = max(1, min(per, (1 << 26) // (tokens * dstate)))
    for lo in [g * per + k for g in range(groups) for k in range(0, per, width)]:
        g = lo // per
        ch = slice(lo, min(lo + width, (g + 1) * per))
        x = flat(s["delta"])[:, ch].double() + s["delta_bias"][ch].double()
        d = torch.logaddexp(x, torch.zeros_like(x))
        u = flat(s["u"])[:, ch].double()
        a = torch.exp(d.unsqueeze(-1) * s["A"][ch].double())
        b = (d * u).unsqueeze(-1) * flat(s["B"])[:, g].double().unsqueeze(1)
        if s["state"] is not None:
            start = s["state"][:, ch] if s["slots"] is None else s["state"][s["slots"].long()][:, ch]
            start = start.double()
            if s["live"] is not None:
                start = start * (s["live"] != 0).double().view(-1, 1, 1)
            b[first] += a[first] * start
        a[first] = 0
        k = 1
        while k < s["longest"]:
            b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
            a = torch.cat([a[:k], a[k:] * a[:-k]])
            k *= 2
        ends[:, ch] = b[last]
        v = torch.einsum("tdn,tn->td", b, flat(s["C"])[:, g].double()) + s["D"][ch].double() * u
        if s["z"] is not None:
            zz = flat(s["z"])[:, ch].double()
            v = v * zz * torch.sigmoid(zz)
        y[:, ch] = v
    pool = _states64(s, ends)
    y = y.reshape(s["u"].shape)
    return y if pool is None else (y, pool)


def _exact_token(s):
    c = s["case"]
    per = c["dim"] // c["groups"]
    pool = s["state"].double()
    y = torch.empty(s["u"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        slot = b if s["slots"] is None else int(s["slots"][b])
        x = s["delta"][b].double() + s["delta_bias"].double()
        d = torch.logaddexp(x, torch.zeros_like(x))
        u = s["u"][b].double()
        h = pool[slot].reshape(c["groups"], per, -1) * torch.exp(d.unsqueeze(-1) * s["A"].double()).reshape(
            c["groups"], per, -1) + torch.einsum("gp,gn->gpn", (d * u).reshape(c["groups"], per), s["B"][b].double())
        v = torch.einsum("gpn,gn->gp", h, s["C"][b].double()).reshape(-1) + s["D"].double() * u
        if s["z"] is not None:
            zz = s["z"][b].double()
            v = v * zz * torch.sigmoid(zz)
        pool[slot] = h.reshape(c["dim"], -1)
        y[b] = v
    return y, pool


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "float32" else 2
    dim = case["dim"]
    if op == "conv":
        w, n = case["width"], case["tokens"] * dim
        states = {"none": 0, "rows": 2, "pool": 1.5}[case["state"]] * case["units"] * dim * (w - 1) * size
        return {"bytes": 2 * n * size + states + dim * (w + int(case["bias"])) * 4,
                "flops": n * (2 * w + (4 if case["silu"] else 0))}
    if op == "conv_token":
        w, n = case["width"], case["batch"] * dim
        return {"bytes": 2 * n * size + 2 * n * (w - 1) * size + dim * (w + int(case["bias"])) * 4,
                "flops": n * (2 * w + (4 if case["silu"] else 0))}
    dstate = case["dstate"]
    params = dim * (dstate + 2) * 4
    rows = case["tokens"] if op == "scan" else case["batch"]
    io = rows * (dim * (4 if case["gate"] else 3) + 2 * case["groups"] * dstate) * size
    states = {"none": 0, "rows": 2, "pool": 1.5}[case["state"]] * case["units"] if op == "scan" else 2 * rows
    # per state and token: delta A, its exponential, delta u B, and two multiply-adds; per channel the softplus,
    # the skip and the gate
    return {"bytes": io + states * dim * dstate * 4 + params,
            "flops": rows * dim * (7 * dstate + 8 + (5 if case["gate"] else 0))}
