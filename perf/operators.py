"""The operators around an 8-bit recogniser, as they are measured: the linear map in 8-bit integers, the step between two
blocks (norm after, gate, residual scale, norm before) and the choice of a beam search with its states.

`listed()` and `draw()` give cases, `prepare()` what a program has in hand before the call, `run()` one pass - by the
framework's kernels where `own` is true, by elementary torch operations in 32 bits where it is false - and `exact()` the
same outputs in 64 bits. Sizes are those of the FastConformer encoder and the TDT joint (width 1024, inner width 4096,
joint 640, 1024 labels + blank + 5 durations, 125 frames for a clip of 10 s, 256 clips) and generic ones around them.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_PACKAGE = Path("kea-kernels_b200")
# Logits lie on a grid of 2^-10, and candidates of different beams that are nearer than this are not asked for: the
# choice between two that differ by less than a 32-bit rounding of the sums would say nothing.
_GRID, _APART = 1024.0, 2e-4


def _lowbit():
    if str(_PACKAGE.resolve()) not in sys.path:
        sys.path.insert(0, str(_PACKAGE.resolve()))
    from kea_kernels import lowbit
    return lowbit


# ---- cases ------------------------------------------------------------------------------------------------------

def _linear(name, m, n, k, out, bias=True, silu=False, residual=0.0):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "out": out, "bias": bias, "silu": silu,
            "residual": residual}


def _block(name, clips, frames, dim, stream, inner, post, pre, gate, act, scale):
    return {"name": name, "op": "block", "clips": clips, "frames": frames, "dim": dim, "stream": stream,
            "inner": inner, "post": post, "pre": pre, "gate": gate, "act": act, "scale": scale}


def _block8(name, clips, frames, dim, n, out, post, gate, act, scale, silu):
    return {"name": name, "op": "block8", "clips": clips, "frames": frames, "dim": dim, "n": n, "out": out,
            "post": post, "pre": "layer", "gate": gate, "act": act, "scale": scale, "silu": silu,
            "stream": "float32", "inner": "float32"}


def _beam(name, clips, beams, vocab, extra, dtype, ended, layers, hidden, state):
    return {"name": name, "op": "beam", "clips": clips, "beams": beams, "vocab": vocab, "extra": extra,
            "dtype": dtype, "ended": ended, "layers": layers, "hidden": hidden, "state": state}


def listed():
    return [
        # one frame through FF-up: what a streaming recogniser issues per frame, latency alone
        _linear("linear frame", 1, 4096, 1024, "float16"),
        # FF-down of one 10 s clip, with its half-step skip connection
        _linear("linear clip", 125, 1024, 4096, "float32", residual=0.5),
        # the joint's output layer over 8 hypotheses of one clip's frames: 1024 labels + blank + 5 durations
        _linear("linear joint", 1000, 1030, 640, "float32"),
        # FF-up of 256 clips
        _linear("linear batch", 32000, 4096, 1024, "float16", silu=True),
        # the prediction state of 8 hypotheses, gated by the last label's embedding
        _block("block beam", 1, 8, 640, "float32", "float32", "layer", "layer", "token", "sigmoid", 1.0),
        # between two macaron halves of 256 clips: half step, a learned gate per channel
        _block("block batch", 256, 125, 1024, "float32", "float32", "layer", "layer", "channel", "none", 0.5),
        # rows of odd width in 16 bits, one gate per clip, root-mean-square norms
        _block("block odd", 24, 501, 1001, "float32", "bfloat16", "rms", "rms", "clip", "none", 1.0),
        # the same step of one clip, straight into the next 8-bit projection
        _block8("block8 clip", 1, 125, 1024, 4096, "float16", "layer", "channel", "none", 0.5, True),
        # and of 64 clips
        _block8("block8 batch", 64, 125, 1024, 4096, "float16", "layer", "token", "sigmoid", 0.5, True),
        # one search step of one clip: 4 hypotheses, rows of the joint's output, two layers of LSTM state
        _beam("beam clip", 1, 4, 1025, 5, "float32", False, 4, 640, "float32"),
        # one search step of 256 clips of which some hypotheses have ended
        _beam("beam batch", 256, 8, 1025, 5, "float32", True, 4, 640, "float32"),
        # a large vocabulary in 16 bits, wider state
        _beam("beam words", 32, 8, 131072, 0, "bfloat16", True, 8, 4096, "float16"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "block", "block8", "beam", "beam"])
    types = ["float32", "float16", "bfloat16"]
    if op == "linear":
        m, n, k = _log_int(rng, 1, 16000), _log_int(rng, 33, 4096), _log_int(rng, 48, 4096)
        residual = rng.choice([0.0, 0.0, 0.5, 1.0])
        case = _linear("", m, n, k, rng.choice(types), rng.random() < 0.7, rng.random() < 0.3 and not residual, residual)
    elif op == "block":
        frames, dim = _log_int(rng, 1, 1500), _log_int(rng, 64, 4096)
        clips = _log_int(rng, 1, max(1, min(256, 32_000_000 // (frames * dim))))
        case = _block("", clips, frames, dim, rng.choice(types), rng.choice(types), rng.choice(["none", "layer", "rms"]),
                      rng.choice(["none", "layer", "rms"]), rng.choice(["none", "channel", "clip", "token"]),
                      rng.choice(["none", "sigmoid"]), rng.choice([0.5, 1.0]))
    elif op == "block8":
        frames, dim, n = _log_int(rng, 1, 500), _log_int(rng, 64, 2048), _log_int(rng, 64, 4096)
        clips = _log_int(rng, 1, max(1, min(64, 8_000_000 // (frames * dim))))
        case = _block8("", clips, frames, dim, n, rng.choice(["float16", "bfloat16"]), rng.choice(["none", "layer", "rms"]),
                       rng.choice(["none", "channel", "clip", "token"]), rng.choice(["none", "sigmoid"]),
                       rng.choice([0.5, 1.0]), rng.random() < 0.5)
    else:
        beams, vocab = _log_int(rng, 1, 16), _log_int(rng, 40, 131072)
        clips = _log_int(rng, 1, max(1, min(256, 30_000_000 // (beams * vocab))))
        case = _beam("", clips, beams, vocab, rng.choice([0, 0, 5]), rng.choice(types), rng.random() < 0.5,
                     rng.choice([1, 2, 4]), _log_int(rng, 64, 2048), rng.choice(["float32", "float16"]))
    del case["name"]
    return case


def _bytes(dtype):
    return 4 if dtype == "float32" else 2


def work(case):
    if case["op"] == "beam":
        rows, state = case["clips"] * case["beams"], _bytes(case["state"])
        return {"bytes": rows * (case["vocab"] * _bytes(case["dtype"]) + 2 * case["layers"] * case["hidden"] * state + 16),
                "flops": 3 * rows * case["vocab"]}
    if case["op"] == "linear":
        m, n, k, size = case["m"], case["n"], case["k"], _bytes(case["out"])
        outputs = m * n * size * (2 if case["residual"] else 1)
        return {"bytes": m * k + n * k + 4 * m + 4 * n * (2 if case["bias"] else 1) + outputs, "flops": 2 * m * n * k}
    rows, dim = case["clips"] * case["frames"], case["dim"]
    inner, stream = _bytes(case["inner"]), _bytes(case["stream"])
    gate = {"none": 0, "channel": dim, "clip": case["clips"] * dim, "token": rows * dim}[case["gate"]] * inner
    moved = rows * dim * (2 * stream + inner) + gate
    if case["op"] == "block":
        return {"bytes": moved + rows * dim * inner, "flops": 16 * rows * dim}
    n = case["n"]   # the codes in between may stay on the chip
    return {"bytes": moved + n * dim + 4 * n + rows * n * _bytes(case["out"]), "flops": (16 + 2 * n) * rows * dim}


# ---- what a program has before the call ----------------------------------------------------------------------------

def _codes(rows, k, gen):
    """Rows of a normal distribution in 8 bits with one scale each, as a quantizer leaves them: (codes, scales). Rows are
    held 16-byte aligned."""
    x = torch.randn(rows, k, generator=gen, device="cuda")
    scale = x.abs().amax(1).clamp_min(1e-30) / 127.0
    codes = torch.zeros(rows, -(-k // 16) * 16, device="cuda", dtype=torch.int8)
    codes[:, :k] = torch.round(x / scale[:, None]).to(torch.int8)
    return codes[:, :k], scale


def _weights(state, n, k, gen, bias):
    state["w"], scale = _codes(n, k, gen)
    state["alpha"] = scale / math.sqrt(k)
    state["bias"] = 0.1 * torch.randn(n, generator=gen, device="cuda") if bias else None


def _norm(kind, dim, gen):
    if kind == "none":
        return None
    module = torch.nn.LayerNorm(dim, device="cuda") if kind == "layer" else torch.nn.RMSNorm(dim, eps=1e-6, device="cuda")
    module.requires_grad_(False)
    module.weight.copy_(1.0 + 0.1 * torch.randn(dim, generator=gen, device="cuda"))
    if kind == "layer":
        module.bias.copy_(0.05 * torch.randn(dim, generator=gen, device="cuda"))
    return module


def _candidates(logits, scores, ended, end):
    """Every continuation's score in 64 bits, [clips, beams * vocab]."""
    x = logits.double()
    x = x - x.exp().sum(-1, keepdim=True).log()   # logits stay far inside the range of exp in 64 bits
    x += scores.double()[..., None]
    if ended is not None:
        x.masked_fill_(ended[..., None], -math.inf)
        x[..., end] = torch.where(ended, scores.double(), x[..., end])
    return x.flatten(1)


def _prepare_beam(case, gen):
    clips, beams, vocab = case["clips"], case["beams"], case["vocab"]
    full = 2.0 * torch.randn(clips, beams, vocab + case["extra"], generator=gen, device="cuda")
    peaks = torch.randint(0, vocab, (clips, beams, 6), generator=gen, device="cuda")   # what the model believes in
    full.scatter_add_(2, peaks, 3.0 + 6.0 * torch.rand(clips, beams, 6, generator=gen, device="cuda"))
    logits = (torch.round(full * _GRID) / _GRID).to(_DTYPES[case["dtype"]])[..., :vocab]
    end = vocab - 1
    ended = torch.rand(clips, beams, generator=gen, device="cuda") < 0.2 if case["ended"] else None
    scores = torch.empty(clips, beams, device="cuda")
    first = torch.arange(clips, device="cuda") % 16 == 15   # clips at their first frame: one hypothesis so far
    loose = torch.ones(clips, dtype=torch.bool, device="cuda")
    for _ in range(40):   # other scores for the clips whose choice would hang on a rounding
        new = -20.0 * torch.rand(clips, beams, generator=gen, device="cuda")
        new[first, 1:] = -math.inf
        scores = torch.where(loose[:, None], new, scores)
        best, at = _candidates(logits, scores, ended, end).topk(min(beams * vocab, beams + 1), 1)
        near = (best[:, :-1] - best[:, 1:] < _APART) & (at[:, :-1] // vocab != at[:, 1:] // vocab)
        loose = near.any(1)
        if not bool(loose.any()):
            break
    states = [torch.randn(clips, beams, case["hidden"], generator=gen, device="cuda").to(_DTYPES[case["state"]])
              for _ in range(case["layers"])]
    return {"logits": logits, "scores": scores, "ended": ended, "end": end, "states": states}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "beam":
        return state | _prepare_beam(case, gen)
    if case["op"] == "linear":
        m, n = case["m"], case["n"]
        state["q"], state["qs"] = _codes(m, case["k"], gen)
        _weights(state, n, case["k"], gen, case["bias"])
        out = _DTYPES[case["out"]]
        state["skip"] = torch.randn(m, n, generator=gen, device="cuda").to(out) if case["residual"] else None
        return state
    shape, dim = (case["clips"], case["frames"]), case["dim"]
    inner = _DTYPES[case["inner"]]
    state["x"] = (2.0 * torch.randn(*shape, dim, generator=gen, device="cuda")).to(_DTYPES[case["stream"]])
    spread = 0.3 + torch.rand(*shape, 1, generator=gen, device="cuda")
    state["y"] = (0.1 + spread * torch.randn(*shape, dim, generator=gen, device="cuda")).to(inner)
    of = {"none": None, "channel": (dim,), "clip": (case["clips"], dim), "token": (*shape, dim)}[case["gate"]]
    state["g"] = None if of is None else (0.5 + 0.5 * torch.randn(*of, generator=gen, device="cuda")).to(inner)
    state["after"], state["before"] = _norm(case["post"], dim, gen), _norm(case["pre"], dim, gen)
    if case["op"] == "block8":
        _weights(state, case["n"], dim, gen, True)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------

def _plain_product(q, qs, state):
    y = (q.float() @ state["w"].float().t()) * qs[:, None] * state["alpha"]
    if state["bias"] is not None:
        y = y + state["bias"]
    return y / (1.0 + torch.exp(-y)) if state["silu"] else y


def _plain_norm(x, module):
    if module is None:
        return x
    if isinstance(module, torch.nn.LayerNorm):
        x = x - x.mean(-1, keepdim=True)
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + module.eps) * module.weight + module.bias
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + module.eps) * module.weight


def _plain_block(state):
    r = _plain_norm(state["y"].float(), state["after"])
    if state["g"] is not None:
        g = state["g"].float()
        g = 1.0 / (1.0 + torch.exp(-g)) if state["act"] == "sigmoid" else g
        r = r * (g[:, None] if state["gate"] == "clip" else g)
    r = state["x"].float() + state["scale"] * r
    return r, _plain_norm(r, state["before"])


def _plain_beam(state):
    x, scores, ended, end = state["logits"].float(), state["scores"], state["ended"], state["end"]
    clips, beams, vocab = x.shape
    top = x.amax(-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))) + scores[..., None]
    if ended is not None:
        x = torch.where(ended[..., None], torch.full_like(x, -math.inf), x)
        x[..., end] = torch.where(ended, scores, x[..., end])
    best, at = torch.sort(x.flatten(1), dim=1, descending=True, stable=True)   # equal ones: the lowest index first
    best, at = best[:, :beams], at[:, :beams]
    parents, tokens = (at // vocab).int(), (at % vocab).int()
    row = torch.arange(clips, device=x.device)[:, None]
    out = {"scores": best, "parents": parents, "tokens": tokens, "states": [s[row, parents] for s in state["states"]]}
    if ended is not None:
        out["ended"] = ended[row, parents] | (tokens == end)
    return out


def _plain(state):
    if state["op"] == "beam":
        return _plain_beam(state)
    if state["op"] == "linear":
        y = _plain_product(state["q"], state["qs"], state)
        if state["residual"]:
            y = state["skip"].float() + state["residual"] * y
        return y.to(_DTYPES[state["out"]])
    r, h = _plain_block(state)
    if state["op"] == "block":
        return {"stream": r.to(state["x"].dtype), "inner": h.to(state["y"].dtype)}
    h = h.flatten(0, 1)
    scale = (h.abs().amax(1) / 127.0).clamp_min(1e-30)
    y = _plain_product(torch.round(h / scale[:, None]), scale, state)
    return {"stream": r.to(state["x"].dtype), "out": y.to(_DTYPES[state["out"]])}


def run(state):
    if not own:
        return _plain(state)
    lowbit = _lowbit()
    if state["op"] == "beam":
        step = lowbit.beam_select(state["logits"], state["scores"], ended=state["ended"], end=state["end"])
        out = {"scores": step.scores, "parents": step.parents, "tokens": step.tokens,
               "states": lowbit.beam_reorder(state["states"], step.parents)}
        if state["ended"] is not None:
            out["ended"] = step.ended
        return out
    if state["op"] == "linear":
        return lowbit.int8_linear(state["q"], state["qs"], state["w"], state["alpha"], state["bias"],
                                  silu=state["silu"], residual=state["skip"], residual_scale=state["residual"],
                                  dtype=_DTYPES[state["out"]])
    options = {"post_norm": state["after"], "gate": state["g"], "gate_act": state["act"], "scale": state["scale"],
               "pre_norm": state["before"]}
    if state["op"] == "block":
        r, h = lowbit.residual_norm(state["x"], state["y"], **options)
        return {"stream": r, "inner": h}
    r, q, qs = lowbit.residual_norm_quantized(state["x"], state["y"], **options)
    y = lowbit.int8_linear(q, qs, state["w"], state["alpha"], state["bias"], silu=state["silu"],
                           dtype=_DTYPES[state["out"]])
    return {"stream": r, "out": y}


# ---- the same in 64 bits -----------------------------------------------------------------------------------------

def _exact_map(codes, scales, state):
    total = torch.einsum("mk,nk->mn", codes.double(), state["w"].double())
    total = torch.einsum("mn,m,n->mn", total, scales.double(), state["alpha"].double())
    if state["bias"] is not None:
        total += state["bias"].double()
    return total * torch.sigmoid(total) if state["silu"] else total


def _exact_norm(x, module):
    if module is None:
        return x
    weight, bias = module.weight.double(), getattr(module, "bias", None)
    centre = x.mean(-1, keepdim=True) if isinstance(module, torch.nn.LayerNorm) else 0.0
    spread = ((x - centre) ** 2).sum(-1, keepdim=True) / x.shape[-1]
    out = weight * (x - centre) / (spread + module.eps).sqrt()
    return out if bias is None else out + bias.double()


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "beam":
        every = _candidates(state["logits"], state["scores"], state["ended"], state["end"])
        best = every.topk(case["beams"], 1).values
        out = {"scores": best, "parents": None, "tokens": None, "states": [None] * case["layers"]}
        return out if state["ended"] is None else out | {"ended": None}
    if case["op"] == "linear":
        y = _exact_map(state["q"], state["qs"], state)
        return y if state["skip"] is None else y * case["residual"] + state["skip"].double()
    step = _exact_norm(state["y"].double(), state["after"])
    if state["g"] is not None:
        g = state["g"].double()
        g = g.sigmoid() if case["act"] == "sigmoid" else g
        step = step * g.view(case["clips"], 1, -1) if case["gate"] == "clip" else step * g
    r = step.mul(case["scale"]).add(state["x"].double())
    h = _exact_norm(r, state["before"])
    if case["op"] == "block":
        return {"stream": r, "inner": h}
    h = h.reshape(-1, case["dim"])
    scales = torch.clamp(h.abs().max(1).values / 127.0, min=1e-30)
    return {"stream": r, "out": _exact_map((h / scales[:, None]).round(), scales, state)}
