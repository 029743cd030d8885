"""Measured cases of the gated linear recurrence and of layer norm, forward and backward.

Five operators carry a gated recurrent layer through training and serving: the
recurrence over long or packed sequences (GatedRecurrenceFn), its backward pass
(GatedRecurrenceGradFn), its form for single tokens over a pool of states
(GatedRecurrenceUpdateFn), and the norm that stands before and behind the layer
with the residual sum it is taken of (LayerNormFn), with its backward pass and
the reduction of the weights' gradients (LayerNormGradFn).
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
EPS = 1e-5
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
        # The benchmark configuration's batch (8 x 2048 tokens, 4096 channels) in a training step's forward pass.
        dict(name="scan_batch", op="scan", dtype="bfloat16", packed=False, units=8, tokens=16384, dim=4096, bound=False,
             state="none"),
        # A prefill step of a server: ragged prompts packed into one row, some continuing a cached state, all states
        # in a pool of slots; the layer's channels have lower bounds of their own.
        dict(name="scan_prompts_packed", op="scan", dtype="bfloat16", packed=True, units=24, tokens=16384, dim=4096,
             bound=True, state="pool"),
        # One long document: few channel rows, a long axis.
        dict(name="scan_long_document", op="scan", dtype="bfloat16", packed=False, units=1, tokens=32768, dim=2048,
             bound=False, state="rows"),
        # A small model in float32, odd length and width, states given and returned.
        dict(name="scan_small_odd", op="scan", dtype="float32", packed=False, units=2, tokens=514, dim=63, bound=True,
             state="rows"),
        # The training step's backward pass, with the gradient of the lower bounds.
        dict(name="grad_batch", op="scan_grad", dtype="bfloat16", packed=False, units=8, tokens=16384, dim=4096,
             bound=True, state="none"),
        # A small model's backward pass in float32 over packed sequences, through the states.
        dict(name="grad_packed_odd", op="scan_grad", dtype="float32", packed=True, units=3, tokens=514, dim=63,
             bound=True, state="rows"),
        # One sequence decoding one token: latency.
        dict(name="token_single", op="token", dtype="bfloat16", batch=1, dim=4096, bound=True, slots=0),
        # A full decode batch over a pool of slots.
        dict(name="token_batch", op="token", dtype="float16", batch=256, dim=4096, bound=True, slots=320),
        # The norm before a layer in a training step: the residual sum and its layer norm, statistics kept.
        dict(name="norm_batch", op="norm", dtype="bfloat16", rows=16384, dim=4096, rms=False, bias=True, residual=True,
             stats=True),
        # The same before a layer of one decoding sequence, without mean and bias: latency.
        dict(name="norm_single", op="norm", dtype="bfloat16", rows=1, dim=4096, rms=True, bias=False, residual=True,
             stats=False),
        # The training step's backward pass, the residual stream's gradient added.
        dict(name="norm_grad_batch", op="norm_grad", dtype="bfloat16", rows=16384, dim=4096, rms=False, bias=True,
             residual=True),
        # A small model's in float32, odd sizes.
        dict(name="norm_grad_odd", op="norm_grad", dtype="float32", rows=514, dim=1001, rms=True, bias=False,
             residual=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _round_dim(rng, n):
    """Most models' widths are multiples of 64; some are not."""
    return max(64, n // 64 * 64) if rng.random() < 0.7 else n


def draw(rng):
    op = rng.choice(["scan", "scan", "scan_grad", "scan_grad", "token", "norm", "norm_grad"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    size = 4 if dtype == "float32" else 2
    dim = _round_dim(rng, _log_int(rng, 48, 8192))
    if op in ("scan", "scan_grad"):
        most = (1 << 26) * 2 // size // dim
        packed = rng.random() < 0.5
        tokens = _log_int(rng, 1, min(32768, most))
        units = _log_int(rng, 1, max(1, min(64, tokens)))
        if not packed:
            tokens = max(1, tokens // units) * units
        return dict(op=op, dtype=dtype, packed=packed, units=units, tokens=tokens, dim=dim, bound=rng.random() < 0.6,
                    state=rng.choice(["none", "rows", "pool"] if op == "scan" else ["none", "rows"]))
    if op == "token":
        batch = _log_int(rng, 1, 1024)
        return dict(op=op, dtype=dtype, batch=batch, dim=dim, bound=rng.random() < 0.6,
                    slots=rng.choice([0, batch + rng.randint(0, 64)]))
    rows = _log_int(rng, 1, min(65536, (1 << 26) * 2 // size // dim))
    case = dict(op=op, dtype=dtype, rows=rows, dim=dim, rms=rng.random() < 0.5, bias=rng.random() < 0.5,
                residual=rng.random() < 0.6)
    if op == "norm":
        case["stats"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------ inputs


class _Maker:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) * 7919 + 29)

    def normal(self, shape, dtype=torch.float32, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std + mean).to(dtype)

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


def _gates(m, shape, dtype):
    """Logits of the share that a channel keeps: most remember tens of tokens, some hundreds, some forget at once."""
    return m.normal(shape, dtype, 1.5, 2.5)


def prepare(case, seed):
    m, op, dt = _Maker(seed), case["op"], DTYPES[case["dtype"]]
    s, dim = {"case": case}, case["dim"]
    if op in ("norm", "norm_grad"):
        rows = case["rows"]
        s["weight"] = m.normal((dim,), std=0.1, mean=1.0)
        s["bias"] = m.normal((dim,), std=0.1) if case["bias"] else None
        # channels differ in scale and offset, as activations do
        scale, offset = torch.exp(m.normal((dim,), std=0.5)), m.normal((dim,), std=0.5)
        x = m.normal((rows, dim)) * scale + offset
        if op == "norm":
            s["x"] = x.to(dt)
            s["residual"] = m.normal((rows, dim), dt, 2.0) if case["residual"] else None
            return s
        s["x"] = x.to(dt)
        s["dy"] = m.normal((rows, dim), dt, 0.1)
        s["dres"] = m.normal((rows, dim), dt, 0.1) if case["residual"] else None
        v = s["x"].float()  # what the forward pass kept
        mean = torch.zeros((rows, 1), device="cuda") if case["rms"] else v.mean(1, keepdim=True)
        s["stats"] = torch.cat([mean, torch.rsqrt(((v - mean) ** 2).mean(1, keepdim=True) + EPS)], 1)
        return s
    s["bound"] = m.uniform((dim,), 0.0, 0.95) if case["bound"] else None
    if op == "token":
        batch = case["batch"]
        n = case["slots"] or batch
        s["x"], s["f"] = m.normal((batch, dim), dt), _gates(m, (batch, dim), dt)
        s["state"] = m.normal((n, dim), std=0.5)
        s["slots"] = m.perm(n)[:batch].to(torch.int32) if case["slots"] else None
        return s
    cu, units = _offsets(m, case), case["units"]
    shape = (1, case["tokens"], dim) if case["packed"] else (units, case["tokens"] // units, dim)
    s["x"], s["f"] = m.normal(shape, dt), _gates(m, shape, dt)
    s["state"] = s["slots"] = s["live"] = None
    if case["state"] == "rows":
        s["state"] = m.normal((units, dim), std=0.5)
    elif case["state"] == "pool":  # about half of the sequences begin anew
        s["state"] = m.normal((units + 16, dim), std=0.5)
        s["slots"] = m.perm(units + 16)[:units].to(torch.int32)
        s["live"] = (m.uniform((units,), 0, 1) < 0.5).to(torch.int32)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    s["longest"] = max(b - a for a, b in zip(cu, cu[1:]))
    if op == "scan_grad":
        s["dy"] = m.normal(shape, dt, 0.1)
        s["dlast"] = m.normal((units, dim), std=0.1) if case["state"] == "rows" else None
        s["y"] = _plain_recurrence(s)[0]  # the forward pass's output, which a training step keeps
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    op = s["case"]["op"]
    if own:
        return {"scan": _own_scan, "scan_grad": _own_scan_grad, "token": _own_token, "norm": _own_norm,
                "norm_grad": _own_norm_grad}[op](s)
    return {"scan": _plain_scan, "scan_grad": _plain_scan_grad, "token": _plain_token, "norm": _plain_norm,
            "norm_grad": _plain_norm_grad}[op](s)


def _own_scan(s):
    c = s["case"]
    return _package().GatedRecurrenceFn(s["x"], s["f"], s["bound"], s["state"], s["cu"] if c["packed"] else None,
                                        s["slots"], s["live"], output_final_state=int(c["state"] != "none"))


def _own_scan_grad(s):
    c = s["case"]
    grads = _package().GatedRecurrenceGradFn(s["dy"], s["x"], s["f"], s["y"], s["bound"], s["state"],
                                             s["cu"] if c["packed"] else None, s["dlast"])
    return [g for g in grads if g is not None]


def _own_token(s):
    return _package().GatedRecurrenceUpdateFn(s["x"], s["f"], s["bound"], s["state"], s["slots"])


def _own_norm(s):
    c = s["case"]
    return _package().LayerNormFn(s["x"], s["weight"], s["bias"], s["residual"], eps=EPS, rms=int(c["rms"]),
                                  output_stats=int(c["stats"]))


def _own_norm_grad(s):
    c = s["case"]
    grads = _package().LayerNormGradFn(s["dy"], s["x"], s["weight"], s["stats"], s["dres"], rms=int(c["rms"]),
                                       output_bias_grad=int(c["bias"]))
    return [g for g in grads if g is not None]


def _shares(f, bound):
    """The share kept, a = bound + (1 - bound) sigmoid(f), and the share taken up, 1 - a without its cancellation."""
    f = f.float()
    rest = 1.0 if bound is None else 1 - bound
    take = rest / (1 + torch.exp(f))
    keep = rest / (1 + torch.exp(-f))
    return keep if bound is None else bound + keep, take


def _start_rows(s):
    """The states that the sequences start from (zeros where there are none)."""
    units, dim = s["case"]["units"], s["case"]["dim"]
    if s["state"] is None:
        return torch.zeros((units, dim), device="cuda")
    rows = s["state"] if s["slots"] is None else s["state"][s["slots"].long()]
    if s["live"] is not None:
        rows = torch.where(s["live"].view(-1, 1) != 0, rows, torch.zeros_like(rows))
    return rows


def _steps(s, width, back=False):
    """Blocks of steps of all sequences at once: the tokens' places [steps, units] and which of them exist."""
    cu = s["cu"].long()
    step = max(1, min(s["longest"], (1 << 25) // width))
    starts = range(0, s["longest"], step)
    for t0 in (reversed(starts) if back else starts):
        t = torch.arange(t0, min(t0 + step, s["longest"]), device="cuda").view(-1, 1)
        at = cu[:-1].view(1, -1) + t
        inside = at < cu[1:].view(1, -1)
        yield torch.where(inside, at, torch.zeros_like(at)), inside


def _plain_recurrence(s):
    dim, units = s["case"]["dim"], s["case"]["units"]
    x, f = s["x"].reshape(-1, dim), s["f"].reshape(-1, dim)
    h = _start_rows(s)
    out = torch.empty_like(x)
    for at, inside in _steps(s, units * dim):
        a, take = _shares(f[at], s["bound"])
        b = take * x[at].float()
        a = torch.where(inside.unsqueeze(-1), a, torch.ones_like(a))
        b = torch.where(inside.unsqueeze(-1), b, torch.zeros_like(b))
        for i in range(a.shape[0]):
            h = torch.addcmul(b[i], a[i], h, out=b[i])
        out[at[inside]] = b[inside].to(out.dtype)
        h = h.clone()
    return out.reshape(s["x"].shape), h


def _plain_scan(s):
    y, h = _plain_recurrence(s)
    if s["state"] is None:
        return y
    if s["slots"] is None:
        return y, h
    s["state"][s["slots"].long()] = h
    return y, s["state"]


def _plain_scan_grad(s):
    dim, units = s["case"]["dim"], s["case"]["units"]
    flat = lambda v: v.reshape(-1, dim)  # noqa: E731
    dy, x, f, y = flat(s["dy"]), flat(s["x"]), flat(s["f"]), flat(s["y"])
    cu = s["cu"].long()
    start = _start_rows(s)
    c = torch.zeros((units, dim), device="cuda") if s["dlast"] is None else s["dlast"]  # a_(t+1) times the state's gradient
    dx, df = torch.empty_like(x), torch.empty_like(f)
    dbound = torch.zeros(dim, dtype=torch.float64, device="cuda")
    for at, inside in _steps(s, units * dim, back=True):
        mask = inside.unsqueeze(-1)
        keep, take = _shares(f[at], s["bound"])
        a = torch.where(mask, keep, torch.ones_like(keep))
        g = torch.where(mask, dy[at].float(), torch.zeros_like(a))
        for i in reversed(range(a.shape[0])):
            torch.add(g[i], c, out=g[i])
            c = a[i] * g[i]
        first = at == cu[:-1].view(1, -1)
        before = torch.where(first.unsqueeze(-1), start.unsqueeze(0), y[(at - 1).clamp(min=0)].float())
        da = g * (before - x[at].float())
        sig = 1 / (1 + torch.exp(-f[at].float()))
        dx[at[inside]] = (take * g)[inside].to(dx.dtype)
        df[at[inside]] = (da * take * sig)[inside].to(df.dtype)
        if s["bound"] is not None:
            part = da / (1 + torch.exp(f[at].float()))
            dbound += torch.where(mask, part, torch.zeros_like(part)).sum((0, 1), dtype=torch.float64)
    out = [dx.reshape(s["x"].shape), df.reshape(s["x"].shape)]
    if s["bound"] is not None:
        out.append(dbound.float())
    if s["state"] is not None:
        out.append(c)
    return out


def _plain_token(s):
    old = s["state"] if s["slots"] is None else s["state"][s["slots"].long()]
    a, take = _shares(s["f"], s["bound"])
    new = a * old + take * s["x"].float()
    if s["slots"] is None:
        s["state"].copy_(new)
    else:
        s["state"][s["slots"].long()] = new
    return new.to(s["x"].dtype), s["state"]


def _plain_norm(s):
    c = s["case"]
    kept = s["x"]
    if s["residual"] is not None:  # the residual stream is stored in the activations' type, and its norm taken of that
        kept = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    v = kept.float()
    mean = torch.zeros((c["rows"], 1), device="cuda") if c["rms"] else v.sum(1, keepdim=True) / c["dim"]
    v = v - mean
    rstd = 1 / torch.sqrt((v * v).sum(1, keepdim=True) / c["dim"] + EPS)
    y = v * rstd * s["weight"]
    if s["bias"] is not None:
        y = y + s["bias"]
    out = [y.to(s["x"].dtype)]
    if s["residual"] is not None:
        out.append(kept)
    if c["stats"]:
        out.append(torch.cat([mean, rstd], 1))
    return out if len(out) > 1 else out[0]


def _plain_norm_grad(s):
    c = s["case"]
    dy, mean, rstd = s["dy"].float(), s["stats"][:, :1], s["stats"][:, 1:]
    xhat = (s["x"].float() - mean) * rstd
    g = dy * s["weight"]
    dx = g - xhat * ((g * xhat).sum(1, keepdim=True) / c["dim"])
    if not c["rms"]:
        dx = dx - g.sum(1, keepdim=True) / c["dim"]
    dx = dx * rstd
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    out = [dx.to(s["x"].dtype), (dy * xhat).sum(0, dtype=torch.float64).float()]
    if c["bias"]:
        out.append(dy.sum(0, dtype=torch.float64).float())
    return out


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "scan_grad": _exact_scan_grad, "token": _exact_token, "norm": _exact_norm,
            "norm_grad": _exact_norm_grad}[case["op"]](s)


def _doubled(a, b, longest):
    """h_t = a_t h_(t-1) + b_t along the first axis by doubling: after the steps 1, 2, 4, ... the pair (a_t, b_t)
    composes every step since the sequence's start, where a = 0."""
    k = 1
    while k < longest:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _slices(case):
    width = max(1, min(case["dim"], (1 << 26) // case["tokens"]))
    return [slice(k, min(k + width, case["dim"])) for k in range(0, case["dim"], width)]


def _gate64(s, ch):
    f = s["f"].reshape(s["case"]["tokens"], -1)[:, ch].double()
    low = torch.zeros((), dtype=torch.float64, device="cuda") if s["bound"] is None else s["bound"][ch].double()
    return low + (1 - low) * torch.sigmoid(f), (1 - low) * torch.sigmoid(-f), f


def _start64(s, ch):
    if s["state"] is None:
        return torch.zeros((s["case"]["units"], len(range(*ch.indices(s["case"]["dim"])))), dtype=torch.float64,
                           device="cuda")
    rows = [s["state"][i if s["slots"] is None else int(s["slots"][i])][ch].double()
            * (1.0 if s["live"] is None else float(int(s["live"][i]) != 0)) for i in range(s["case"]["units"])]
    return torch.stack(rows)


def _exact_scan(s):
    c = s["case"]
    bounds = s["cu"].long()
    first, last = bounds[:-1], bounds[1:] - 1
    y = torch.empty((c["tokens"], c["dim"]), dtype=torch.float64, device="cuda")
    for ch in _slices(c):
        a, u, _ = _gate64(s, ch)
        b = u * s["x"].reshape(c["tokens"], -1)[:, ch].double()
        b[first] += a[first] * _start64(s, ch)
        a[first] = 0
        y[:, ch] = _doubled(a, b, s["longest"])
    out = y.reshape(s["x"].shape)
    if s["state"] is None:
        return out
    if s["slots"] is None:
        return out, y[last]
    pool = s["state"].double()
    pool[s["slots"].long()] = y[last]
    return out, pool


def _exact_scan_grad(s):
    c = s["case"]
    n = c["tokens"]
    flat = lambda k, ch: s[k].reshape(n, -1)[:, ch].double()  # noqa: E731
    bounds = s["cu"].long()
    first, last = bounds[:-1], bounds[1:] - 1
    dx, df = (torch.empty((n, c["dim"]), dtype=torch.float64, device="cuda") for _ in range(2))
    dbound = torch.empty(c["dim"], dtype=torch.float64, device="cuda")
    dstart = torch.empty((c["units"], c["dim"]), dtype=torch.float64, device="cuda")
    for ch in _slices(c):
        a, u, f = _gate64(s, ch)
        # in reversed order, G_t = dy_t + a_(t+1) G_(t+1)
        b = flat("dy", ch)
        if s["dlast"] is not None:
            b[last] += s["dlast"][:, ch].double()
        nxt = torch.cat([a[1:], torch.zeros_like(a[:1])])
        nxt[last] = 0
        g = _doubled(nxt.flip(0), b.flip(0), s["longest"]).flip(0)
        prev = torch.cat([torch.zeros_like(g[:1]), flat("y", ch)[:-1]])
        prev[first] = _start64(s, ch)
        da = g * (prev - flat("x", ch))
        dx[:, ch] = u * g
        df[:, ch] = da * u * torch.sigmoid(f)
        dbound[ch] = (da * torch.sigmoid(-f)).sum(0)
        dstart[:, ch] = (a * g)[first]
    out = [dx.reshape(s["x"].shape), df.reshape(s["x"].shape)]
    if s["bound"] is not None:
        out.append(dbound)
    if s["state"] is not None:
        out.append(dstart)
    return out


def _exact_token(s):
    low = 0.0 if s["bound"] is None else s["bound"].double()
    pool, f, x = s["state"].double(), s["f"].double(), s["x"].double()
    y = torch.empty_like(x)
    for b in range(x.shape[0]):
        slot = b if s["slots"] is None else int(s["slots"][b])
        a = low + (1 - low) * torch.sigmoid(f[b])
        pool[slot] = a * pool[slot] + (1 - low) * torch.sigmoid(-f[b]) * x[b]
        y[b] = pool[slot]
    return y, pool


def _exact_norm(s):
    c = s["case"]
    total = s["x"].double()
    kept = total
    if s["residual"] is not None:
        total = total + s["residual"].double()
        kept = total.to(s["x"].dtype).double()
    mean = kept.mean(1) if not c["rms"] else torch.zeros(c["rows"], dtype=torch.float64, device="cuda")
    var = torch.einsum("rd,rd->r", kept - mean.unsqueeze(1), kept - mean.unsqueeze(1)) / c["dim"]
    rstd = (var + EPS) ** -0.5
    y = (kept - mean.unsqueeze(1)) * torch.outer(rstd, s["weight"].double())
    if s["bias"] is not None:
        y = y + s["bias"].double()
    out = [y] + ([total] if s["residual"] is not None else []) + ([torch.stack([mean, rstd], 1)] if c["stats"] else [])
    return out if len(out) > 1 else out[0]


def _exact_norm_grad(s):
    c = s["case"]
    dy, mean, rstd = s["dy"].double(), s["stats"][:, 0].double(), s["stats"][:, 1].double()
    xhat = (s["x"].double() - mean.unsqueeze(1)) * rstd.unsqueeze(1)
    g = dy * s["weight"].double()
    along = torch.einsum("rd,rd->r", g, xhat) / c["dim"]
    dx = g - xhat * along.unsqueeze(1) - (0.0 if c["rms"] else g.mean(1, keepdim=True))
    dx = dx * rstd.unsqueeze(1)
    if s["dres"] is not None:
        dx = dx + s["dres"].double()
    return [dx, torch.einsum("rd,rd->d", dy, xhat)] + ([dy.sum(0)] if c["bias"] else [])


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op, size, dim = case["op"], 4 if case["dtype"] == "float32" else 2, case["dim"]
    if op in ("norm", "norm_grad"):
        n = case["rows"] * dim
        params = dim * 4 * (1 + int(case["bias"]))
        if op == "norm":
            # x and y, with a residual it and the sum; per element the sum, mean, variance, scaling, weight and bias
            return {"bytes": n * size * (4 if case["residual"] else 2) + params + (8 * case["rows"] if case["stats"] else 0),
                    "flops": n * (5 + 2 * (not case["rms"]) + int(case["bias"]) + int(case["residual"]))}
        # dy, x, dx and the residual's gradient; the weights' gradients; per element xhat, both sums, dx, both gradients
        return {"bytes": n * size * (4 if case["residual"] else 3) + params + dim * 4 + 8 * case["rows"],
                "flops": n * (9 + 3 * (not case["rms"]) + int(case["bias"]) + int(case["residual"]))}
    bound = dim * 4 if case["bound"] else 0
    if op == "token":
        n = case["batch"] * dim
        return {"bytes": n * (3 * size + 8) + bound, "flops": n * (8 + 2 * int(case["bound"]))}
    n = case["tokens"] * dim
    row = case["units"] * dim * 4
    if op == "scan":
        # x, f and y; the states; per element both shares (exponential, sum, quotients) and the update
        return {"bytes": 3 * n * size + {"none": 0, "rows": 2, "pool": 1.5}[case["state"]] * row + bound,
                "flops": n * (8 + 2 * int(case["bound"]))}
    # dy, x, f, y, dx and df; states, their gradients in and out; per element the shares, both gradients and the carry
    return {"bytes": 6 * n * size + (3 * row if case["state"] == "rows" else 0) + 2 * bound,
            "flops": n * (14 + 4 * int(case["bound"]))}
