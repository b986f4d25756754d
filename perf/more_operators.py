"""A quantized transformer layer's path to its answer, measured: root-mean-square
norm with the residual's addition (forward, backward, and with an output in 8
bits), rows in 8 bits with a scale each, the product of such rows with 8-bit
weights with bias, activation and residual in its epilogue, and the log
probabilities of given tokens with entropy, top alternatives and their gradient.

`run` makes one pass: in elementary torch operations, or, with `own` set, through
the library's C entry points as a pyneural program calls them, outputs in place.

Definitions.  Norm: h = in + residual, rstd = 1 / sqrt(sum(h^2) / C + eps), out =
h rstd gamma; backward from the saved rstd: w = dy gamma, xh = h rstd, grad = rstd
(w - xh mean(w xh)) + dh, dgamma = sum over rows of dy xh.

8 bits: for a row of values w, a = max |w|, code = 127 w / a rounded to the
nearest whole number, halves away from zero; scale = a / 127.  The norm's codes
are those of its output's row: of w = h gamma, with scale = a rstd / 127.  Codes
are made in 64 bits, since a quotient next to a half decides them.

Linear: out = act(scale[m] wscale[n] sum_k code[m, k] wcode[n, k] + bias[n]) +
residual[m, n]; gelu by tanh, swish(x) = x sigmoid(x).

Log probabilities: z = logits / temperature, lse = log sum exp z, logprob = z_t -
lse, entropy = -sum p log p, and the k largest z - lse with their indices, equal
ones by index; a masked logit (-inf) is no alternative (index -1, -inf).  A
negative token: the row is not used (0, and no alternatives).  Gradient, of
logprob by g and entropy by e: (g (1_t - p) - e p (log p + entropy)) / temperature.
"""

import ctypes
import math
import os
import sys

import torch

own = False

EPS = 1e-6
_F = {"f32": torch.float32, "f64": torch.float64}
_ES = {"f32": 4, "f64": 8}
_GELU = 0.7978845608028654


# ---- the listed cases ------------------------------------------------------------


def listed():
    return [
        # A decode step of one sequence: residual add, norm to 8 bits, and a
        # projection.  The latency of two dependent calls, and 16 MB of weights.
        {"name": "token_projection", "kind": "norm_linear", "rows": 1, "k": 4096, "n": 4096, "act": "none",
         "bias": False, "dtype": "f32"},
        # The same for a serving batch into the wide half of a feed-forward layer.
        {"name": "decode_feed_forward", "kind": "norm_linear", "rows": 64, "k": 4096, "n": 16384, "act": "gelu",
         "bias": True, "dtype": "f32"},
        # A prefill of 8192 tokens through it.
        {"name": "prefill_feed_forward", "kind": "norm_linear", "rows": 8192, "k": 4096, "n": 16384, "act": "gelu",
         "bias": True, "dtype": "f32"},
        # The way back to the residual stream: activations to 8 bits, the narrow
        # product, and the stream added in its epilogue.
        {"name": "feed_forward_out", "kind": "linear", "rows": 4096, "k": 16384, "n": 4096, "act": "none",
         "bias": True, "residual": True, "dtype": "f32"},
        # Sizes that are no multiple of anything, in double.
        {"name": "odd_linear_f64", "kind": "linear", "rows": 577, "k": 1001, "n": 3001, "act": "swish", "bias": True,
         "residual": True, "dtype": "f64"},
        # The norm in a wide model's training batch, with the residual add.
        {"name": "norm", "kind": "norm", "rows": 16384, "cols": 4096, "residual": True, "dtype": "f32"},
        # Odd rows in double, alone.
        {"name": "odd_norm_f64", "kind": "norm", "rows": 5003, "cols": 1001, "residual": False, "dtype": "f64"},
        # Its gradient in a short sequence's fine-tuning: few rows to reduce over.
        {"name": "small_norm_grad", "kind": "norm_grad", "rows": 197, "cols": 768, "residual": False, "dtype": "f32"},
        # The gradient in the training batch, joined with the residual stream's.
        {"name": "norm_grad", "kind": "norm_grad", "rows": 16384, "cols": 4096, "residual": True, "dtype": "f32"},
        # One sequence's sampled token: its log probability and 20 alternatives.
        {"name": "token_logprobs", "kind": "logprobs", "rows": 1, "vocab": 131072, "top": 20, "temperature": 1.0,
         "masked": 0.0, "dtype": "f32"},
        # A serving batch's, under a grammar that rules tokens out.
        {"name": "decode_logprobs", "kind": "logprobs", "rows": 64, "vocab": 32000, "top": 20, "temperature": 0.8,
         "masked": 0.3, "dtype": "f32"},
        # A policy's training step on sampled tokens, with an entropy term:
        # forward and gradient over a batch with padded rows.
        {"name": "policy_step", "kind": "logprobs_step", "rows": 4096, "vocab": 50257, "temperature": 1.0,
         "dtype": "f32"},
    ]


# ---- drawn cases -----------------------------------------------------------------


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; every other one as it falls
    (mostly odd), the rest rounded to a multiple of 64 as layer widths are."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))
    if rng.random() < 0.5 and v >= 128:
        v = (v + 32) // 64 * 64
    return max(lo, min(max(lo, hi), v))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "linear", "norm_linear", "linear", "norm_linear", "logprobs",
                       "logprobs_step"])
    dtype = "f64" if rng.random() < 0.25 else "f32"
    half = 2 if dtype == "f64" else 1
    if kind in ("norm", "norm_grad"):
        cols = _size(rng, 16, 16384)
        return {"kind": kind, "rows": _size(rng, 1, 67108864 // half // cols), "cols": cols,
                "residual": rng.random() < 0.5, "dtype": dtype}
    if kind in ("linear", "norm_linear"):
        k, n = _size(rng, 64, 16384), _size(rng, 64, 16384)
        most = min(8192 * 4096 * 16384 // (k * n), 67108864 // max(k, n)) // half
        case = {"kind": kind, "rows": _size(rng, 1, max(1, min(8192, most))), "k": k, "n": n,
                "act": rng.choice(["none", "gelu", "swish", "relu"]), "bias": rng.random() < 0.7, "dtype": dtype}
        if kind == "linear":
            case["residual"] = rng.random() < 0.5
        return case
    vocab = _size(rng, 1000, 131072)
    if kind == "logprobs":
        return {"kind": kind, "rows": _size(rng, 1, 16777216 // vocab), "vocab": vocab, "top": rng.randrange(0, 33),
                "temperature": rng.choice([0.6, 1.0, 1.0, 1.3]), "masked": rng.choice([0.0, 0.0, 0.3, 0.95]),
                "dtype": dtype}
    return {"kind": kind, "rows": _size(rng, 16, 134217728 // half // vocab), "vocab": vocab,
            "temperature": rng.choice([0.7, 1.0, 1.0]), "dtype": dtype}


# ---- inputs ----------------------------------------------------------------------


class _Draws:
    """Seeded GPU tensors (the same for the same seed)."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(4000037 + int(seed))

    def normal(self, shape, dtype, std=1.0, mean=0.0):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=dtype).mul_(std).add_(mean)

    def hidden(self, shape, dtype):
        """Hidden states: a few channels with far larger values."""
        x = self.normal(shape, dtype)
        x[:, self.integers((max(1, shape[1] // 200),), 0, shape[1])] *= 20.0
        return x

    def integers(self, shape, lo, hi):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda")

    def share(self, shape, p):
        return torch.rand(shape, generator=self.g, device="cuda") < p


def _weights(r, n, k, dtype):
    """8-bit weights as a checkpoint holds them: codes by output channel, a scale each."""
    w = r.normal((n, k), torch.float32, k ** -0.5)
    a = w.abs().amax(1, keepdim=True)
    return (w * (127.0 / a)).round_().to(torch.int8), (a[:, 0].double() / 127.0).to(dtype)


def _inputs(case, seed):
    """The case's inputs, from the seed alone."""
    r = _Draws(seed)
    kind, T, rows = case["kind"], _F[case["dtype"]], case["rows"]
    d = {}
    if kind in ("norm", "norm_grad"):
        shape = (rows, case["cols"])
        d["x"], d["gamma"] = r.hidden(shape, T), r.normal(shape[1:], T, 0.2, 1.0)
        if kind == "norm" and case["residual"]:
            d["residual"] = r.normal(shape, T, 2.0)
        if kind == "norm_grad":  # x: the normalised rows, with their saved statistic
            d["dy"] = r.normal(shape, T, 0.01)
            d["rstd"] = (d["x"].double().square().mean(1) + EPS).rsqrt().to(T)
            if case["residual"]:
                d["dh"] = r.normal(shape, T, 0.01)
    elif kind in ("linear", "norm_linear"):
        d["x"] = r.hidden((rows, case["k"]), T)
        d["wcode"], d["wscale"] = _weights(r, case["n"], case["k"], T)
        if case["bias"]:
            d["bias"] = r.normal((case["n"],), T, 0.2)
        if kind == "norm_linear":
            d["residual"], d["gamma"] = r.normal((rows, case["k"]), T, 2.0), r.normal((case["k"],), T, 0.2, 1.0)
        elif case["residual"]:
            d["residual"] = r.normal((rows, case["n"]), T, 2.0)
    else:
        shape = (rows, case["vocab"])
        d["logits"] = r.normal(shape, T, 2.5)
        d["tokens"] = r.integers((rows,), 0, case["vocab"])
        likely = r.integers((rows, 4), 0, case["vocab"])
        likely[:, 0] = torch.where(r.share((rows,), 0.7), d["tokens"], likely[:, 0])  # often the likeliest
        d["logits"].scatter_add_(1, likely, r.normal((rows, 4), T, 2.0, 9.0))
        if case.get("masked", 0.0) > 0.0:
            ruled_out = r.share(shape, case["masked"]).scatter_(1, d["tokens"][:, None], False)
            d["logits"].masked_fill_(ruled_out, -math.inf)
        if kind == "logprobs_step":
            d["tokens"].masked_fill_(r.share((rows,), 0.1), -1)  # padding
            d["g"], d["e"] = r.normal((rows,), T, 1.0 / rows), r.normal((rows,), T, 0.01 / rows)
    return d


def _package():
    p = os.path.join(os.getcwd(), "neural-assembly_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import pyneural
    return pyneural


def _outputs(case):
    """The output tensors that a program holds: shapes and types by name."""
    T, rows, kind = _F[case["dtype"]], case["rows"], case["kind"]
    if kind == "norm":
        return {"out": ((rows, case["cols"]), T), "rstd": ((rows,), T),
                **({"hidden": ((rows, case["cols"]), T)} if case["residual"] else {})}
    if kind == "norm_grad":
        return {"grad": ((rows, case["cols"]), T), "dgamma": ((case["cols"],), T)}
    if kind in ("linear", "norm_linear"):
        return {"out": ((rows, case["n"]), T), "scale": ((rows,), T),
                **({"hidden": ((rows, case["k"]), T)} if kind == "norm_linear" else {})}
    o = {"logprob": ((rows,), T), "entropy": ((rows,), T), "lse": ((rows,), T)}
    if kind == "logprobs_step":
        o["grad"] = ((rows, case["vocab"]), T)
    elif case["top"]:
        o["top_ids"], o["top_logprobs"] = ((rows, case["top"]), torch.int64), ((rows, case["top"]), T)
    return o


def prepare(case, seed):
    s = {"case": dict(case), "in": _inputs(case, seed)}
    if own:
        # the tensor handles that a pyneural program holds, on torch's stream, and its output tensors
        pn = _package()
        pn.set_stream(torch.cuda.current_stream().cuda_stream)
        s["out"] = {k: torch.empty(shape, dtype=t, device="cuda") for k, (shape, t) in _outputs(case).items()}
        if "k" in case:  # the rows' codes, between the two calls
            s["codes"] = torch.empty((case["rows"], case["k"]), dtype=torch.int8, device="cuda")
        s["lib"] = pn.core._lib
        wrap = lambda t: pn.Tensor.from_torch(t) if t.is_floating_point() else t  # noqa: E731
        s["t"] = {k: wrap(v) for k, v in s["in"].items()}
        s["t"].update(("out_" + k, wrap(v)) for k, v in s["out"].items())
        s["at"] = {k: v.data_ptr() if isinstance(v, torch.Tensor) else v._ptr for k, v in s["t"].items()}
        s["act"] = pn.nn.ACTIVATIONS[case.get("act", "none")]
    return s


# ---- one pass through the library ------------------------------------------------


def _run_own(s):
    case, lib, t, at = s["case"], s["lib"], s["at"], s["at"].get
    kind = case["kind"]
    rc = 0
    if kind == "norm":
        rc = lib.neural_rms_norm_forward(t["out_out"], at("out_hidden"), t["x"], at("residual"), t["gamma"], EPS,
                                         t["out_rstd"])
    elif kind == "norm_grad":
        rc = lib.neural_rms_norm_backward(t["out_grad"], t["out_dgamma"], t["dy"], at("dh"), t["x"], t["gamma"],
                                          t["rstd"])
    elif kind in ("linear", "norm_linear"):
        codes, k = s["codes"].data_ptr(), case["k"]
        if kind == "linear":
            rc = lib.neural_quantize_rows(codes, k, t["out_scale"], t["x"])
        else:
            rc = lib.neural_rms_norm_forward_q8(codes, k, t["out_scale"], t["out_hidden"], t["x"], t["residual"],
                                                t["gamma"], EPS)
        rc = rc or lib.neural_linear_q8(t["out_out"], codes, k, t["out_scale"], t["wcode"], k, t["wscale"], k,
                                        at("bias"), s["act"], 0.0, at("residual") if kind == "linear" else None)
    else:
        top = case.get("top", 0)
        rc = lib.neural_token_logprobs_forward(t["out_logprob"], t["out_entropy"], t["out_lse"], at("out_top_ids"),
                                               at("out_top_logprobs"), top, t["logits"], t["tokens"],
                                               case["temperature"])
        if kind == "logprobs_step":
            rc = rc or lib.neural_token_logprobs_backward(t["out_grad"], t["g"], t["e"], t["logits"], t["tokens"],
                                                          t["out_lse"], t["out_entropy"], case["temperature"])
    if rc != 0:
        raise RuntimeError("the library returned %d" % rc)
    return s["out"]


# ---- the plain form --------------------------------------------------------------


def _codes(w):
    """(codes as float64, max |w| by row) of rows in 64 bits."""
    a = w.abs().amax(1, keepdim=True)
    q = torch.where(a > 0, w * 127.0 / a, w)
    return torch.sign(q) * torch.floor(q.abs() + 0.5), a


def _act(x, act):
    if act == "relu":
        return x * (x > 0)
    if act == "swish":
        return x / (1.0 + torch.exp(-x))
    if act == "gelu":  # 1 + tanh(z) = 2 / (1 + exp(-2 z))
        return x / (1.0 + torch.exp(-2.0 * _GELU * (x + 0.044715 * x * x * x)))
    return x


def _plain_linear(case, d):
    T = _F[case["dtype"]]
    o = {}
    if case["kind"] == "norm_linear":
        o["hidden"] = d["x"] + d["residual"]
        h = o["hidden"].double()
        codes, a = _codes(h * d["gamma"].double())
        scale = (a[:, 0] / 127.0 / torch.sqrt((h * h).sum(1) / case["k"] + EPS)).to(T)
    else:
        codes, a = _codes(d["x"].double())
        scale = (a[:, 0] / 127.0).to(T)
    y = codes.to(T) @ d["wcode"].to(T).t()
    y = y * scale[:, None] * d["wscale"]
    if case["bias"]:
        y = y + d["bias"]
    y = _act(y, case["act"])
    if case.get("residual"):
        y = y + d["residual"]
    return {"out": y, "scale": scale, **o}


def _plain_logprobs(case, d):
    x = d["logits"] / case["temperature"]
    used = d["tokens"] >= 0
    zero = torch.zeros((), dtype=x.dtype, device=x.device)
    m = x.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    logp = x - lse
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, zero).sum(1)
    logprob = logp.gather(1, d["tokens"].clamp(min=0)[:, None])[:, 0]
    o = {"logprob": torch.where(used, logprob, zero), "entropy": torch.where(used, entropy, zero),
         "lse": torch.where(used, lse[:, 0], zero)}
    if case["kind"] == "logprobs_step":
        at = torch.arange(case["vocab"], device=x.device) == d["tokens"][:, None]
        grad = d["g"][:, None] * (at.to(x.dtype) - p)
        grad = grad - d["e"][:, None] * torch.where(p > 0, p * (logp + entropy[:, None]), zero)
        o["grad"] = torch.where(used[:, None], grad / case["temperature"], zero)
    elif case["top"]:
        ids = torch.sort(d["logits"], dim=1, descending=True, stable=True).indices[:, :case["top"]]
        best = logp.gather(1, ids)
        none = (best == -math.inf) | ~used[:, None]
        o["top_ids"] = torch.where(none, torch.full_like(ids, -1), ids)
        o["top_logprobs"] = torch.where(none, torch.full_like(best, -math.inf), best)
    return o


def run(s):
    if own:
        return _run_own(s)
    case, d = s["case"], s["in"]
    kind = case["kind"]
    if kind in ("linear", "norm_linear"):
        return _plain_linear(case, d)
    if kind in ("logprobs", "logprobs_step"):
        return _plain_logprobs(case, d)
    if kind == "norm":
        h = d["x"] + d["residual"] if case["residual"] else d["x"]
        rstd = 1.0 / torch.sqrt((h * h).sum(1) / case["cols"] + EPS)
        return {"out": h * rstd[:, None] * d["gamma"], "rstd": rstd, **({"hidden": h} if case["residual"] else {})}
    w, xh = d["dy"] * d["gamma"], d["x"] * d["rstd"][:, None]
    grad = d["rstd"][:, None] * (w - xh * ((w * xh).sum(1, keepdim=True) / case["cols"]))
    if case["residual"]:
        grad = grad + d["dh"]
    return {"grad": grad, "dgamma": (d["dy"] * xh).sum(0)}


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    es, rows, kind = _ES[case["dtype"]], case["rows"], case["kind"]
    if kind == "norm":
        n = rows * case["cols"]
        return {"bytes": es * ((4 if case["residual"] else 2) * n + case["cols"] + rows), "flops": 5 * n}
    if kind == "norm_grad":
        n = rows * case["cols"]
        return {"bytes": es * ((4 if case["residual"] else 3) * n + 2 * case["cols"] + rows), "flops": 9 * n}
    if kind in ("linear", "norm_linear"):
        k, n = case["k"], case["n"]
        b = n * k + es * (rows * n + rows * k + n + rows + (n if case["bias"] else 0))
        if kind == "norm_linear":
            b += es * (2 * rows * k + k)
        elif case["residual"]:
            b += es * rows * n
        return {"bytes": b, "flops": 2 * rows * k * n}
    n = rows * case["vocab"]
    if kind == "logprobs_step":  # the gradient needs a whole row's sums first: the logits twice
        return {"bytes": es * (3 * n + 5 * rows) + 8 * rows, "flops": 20 * n}
    return {"bytes": es * (n + 3 * rows) + 8 * rows + (8 + es) * rows * case["top"], "flops": 8 * n}


# ---- the same in 64 bits, from the definitions -------------------------------------


def _exact_codes(v):
    top = v.abs().max(dim=1).values
    ratio = (v / torch.where(top == 0, torch.ones_like(top), top)[:, None]) * 127.0
    down = torch.trunc(ratio)
    return down + torch.trunc(2.0 * (ratio - down)), top


def exact(case, seed):
    d = _inputs(case, seed)
    kind, rows = case["kind"], case["rows"]
    t = {k: v if v.dtype == torch.int64 else v.double() for k, v in d.items()}
    if kind == "norm":
        h = t["x"] + t["residual"] if case["residual"] else t["x"]
        rstd = (h.pow(2).mean(1) + EPS).pow(-0.5)
        o = {"out": torch.mul(torch.mul(h, t["gamma"]), rstd.unsqueeze(1)), "rstd": rstd}
        return {**o, "hidden": h} if case["residual"] else o
    if kind == "norm_grad":
        rstd = t["rstd"].unsqueeze(1)
        w = t["gamma"] * t["dy"]
        along = torch.linalg.vecdot(w, t["x"]).unsqueeze(1) / case["cols"]
        g = rstd * w - rstd.pow(3) * along * t["x"]
        return {"grad": g + t["dh"] if case["residual"] else g, "dgamma": (t["x"] * t["dy"]).t() @ t["rstd"]}
    if kind in ("linear", "norm_linear"):
        o = {}
        if kind == "norm_linear":
            h = (d["x"] + d["residual"]).double()  # codes are of the stored sum
            code, top = _exact_codes(h * t["gamma"])
            o = {"hidden": t["x"] + t["residual"], "scale": top * (h.pow(2).mean(1) + EPS).pow(-0.5) / 127.0}
        else:
            code, top = _exact_codes(t["x"])
            o = {"scale": top / 127.0}
        y = torch.outer(o["scale"], t["wscale"]) * torch.mm(code, t["wcode"].t().contiguous())
        if case["bias"]:
            y += t["bias"]
        if case["act"] == "relu":
            y = torch.clamp(y, min=0.0)
        elif case["act"] == "swish":
            y = y * torch.sigmoid(y)
        elif case["act"] == "gelu":
            y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y.pow(3))))
        return {"out": y + t["residual"] if case.get("residual") else y, **o}
    out = None
    for r0 in range(0, rows, 512):  # a part of the rows at a time
        part = slice(r0, min(rows, r0 + 512))
        z, tok = t["logits"][part] / case["temperature"], t["tokens"][part]
        used = (tok >= 0).double()
        lse = torch.logsumexp(z, 1)
        p = torch.softmax(z, 1)
        entropy = torch.special.entr(p).sum(1)
        here = {"lse": torch.where(tok >= 0, lse, 0.0), "entropy": entropy * used}
        picked = z.gather(1, tok.clamp(min=0).unsqueeze(1)).squeeze(1) - lse
        here["logprob"] = torch.where(tok >= 0, picked, 0.0)
        if kind == "logprobs_step":
            g, e = t["g"][part] * used, t["e"][part] * used
            down = -g.unsqueeze(1) * p + e.unsqueeze(1) * (torch.special.entr(p) - p * entropy.unsqueeze(1))
            down.scatter_add_(1, tok.clamp(min=0).unsqueeze(1), g.unsqueeze(1))
            here["grad"] = down / case["temperature"]
        elif case["top"]:
            order = torch.argsort(-z, dim=1, stable=True)[:, :case["top"]]
            best = z.gather(1, order)
            no = torch.isinf(best) | (tok < 0).unsqueeze(1)
            here["top_ids"] = order.masked_fill(no, -1)
            here["top_logprobs"] = (best - lse.unsqueeze(1)).masked_fill(no, -math.inf)
        out = here if out is None else {k: torch.cat([out[k], v]) for k, v in here.items()}
    order = ["logprob", "entropy", "lse", "grad", "top_ids", "top_logprobs"]
    return {k: out[k] for k in order if k in out}
