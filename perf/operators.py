"""The operators of deep language-model stacks that this framework offers beside its layers, as cases
to be timed: the loss over a large vocabulary with its gradient, the norms around a residual block with
their gradients, and activations kept in 8 bits for the backward pass.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at
the end) or, where ``own`` is true, through the framework's public entry points.  ``exact`` computes the
same outputs in 64 bits.

Vocabulary loss: logits = scale * hidden @ weight.T + bias; loss = logsumexp(logits) - logits[target];
rows whose target is outside the vocabulary are ignored.
Residual norm: new = stream_scale * stream + branch_scale * gate * norm(branch); normed = norm(new).
Packed activations: out = f(x), with x kept as 8-bit codes and one scale for 128 elements of a row.
"""
import math

import torch

own = False

BLOCK = 128          # elements of a row that share a scale
TINY = 2.0 ** -100   # a block with nothing larger is held as zeros
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------ the cases
def _ce(call, rows, width, vocab, dtype, bias=False):
    return dict(op="ce", call=call, rows=rows, width=width, vocab=vocab, dtype=dtype, bias=bias)


def _norm(call, rows, width, dtype, kind="rms", groups=1, post=True, bias=False):
    return dict(op="norm", call=call, rows=rows, width=width, dtype=dtype, kind=kind, groups=groups,
                post=post, bias=bias)


def _pack(call, rows, width, dtype, act):
    return dict(op="pack", call=call, rows=rows, width=width, dtype=dtype, act=act)


def listed():
    cases = {
        # The likelihood of one token while serving: all of the weights are read for one row.
        "ce_score_token": _ce("forward", 1, 1024, 32000, "bf16"),
        # The loss of an evaluation batch: no gradients are wanted.
        "ce_evaluate": _ce("forward", 2048, 1024, 50021, "bf16"),
        # A small network in 32 bits with a bias and with sizes that fit no tile.
        "ce_ragged_f32": _ce("train", 777, 515, 10007, "f32", bias=True),
        # The head of an ordinary training step: loss and gradients.
        "ce_train": _ce("train", 4096, 1024, 50021, "bf16"),
        # The largest head: 8192 tokens against 128000 words.
        "ce_train_large": _ce("train", 8192, 2048, 128000, "bf16"),
        # Norms around a block for one token: launch latency.
        "norm_token": _norm("forward", 1, 2048, "bf16"),
        # The same for a training batch.
        "norm_forward": _norm("forward", 16384, 2048, "bf16"),
        # Gradients of a wide block whose gate differs from sequence to sequence.
        "norm_backward": _norm("backward", 16384, 4096, "bf16", groups=8),
        # Layer norms with biases in 32 bits, odd widths, seven sequences.
        "norm_ragged_f32": _norm("backward", 1001, 1023, "f32", kind="layer", groups=7, bias=True),
        # A small layer's activations kept and restored: launch latency and a short last block.
        "pack_small": _pack("restore", 64, 1000, "f32", "tanh"),
        # A wide layer's activations of a training batch kept and restored.
        "pack_restore": _pack("restore", 16384, 8192, "bf16", "gelu"),
        # The gradient through that layer's activation, with its output for the weight gradient.
        "pack_backward": _pack("backward", 16384, 8192, "bf16", "gelu"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _between(rng, low, high):
    """A whole number of [low, high], spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("ce", "norm", "pack"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if op == "ce":
        top = (8192, 2048, 128000) if dtype == "bf16" else (2048, 1024, 32000)
        rows, width, vocab = _between(rng, 1, top[0]), _between(rng, 64, top[1]), _between(rng, 1000, top[2])
        return _ce(rng.choice(("forward", "train", "train")), rows, width, vocab, dtype, rng.random() < 0.3)
    if op == "norm":
        groups = rng.choice((0, 1, 1, _between(rng, 2, 64)))
        rows, width = _between(rng, 1, 16384), _between(rng, 64, 4096 if dtype == "bf16" else 2048)
        rows = max(1, rows // max(1, groups)) * max(1, groups)
        return _norm(rng.choice(("forward", "backward")), rows, width, dtype, rng.choice(("rms", "layer")),
                     groups, rng.random() < 0.7, rng.random() < 0.4)
    rows, width = _between(rng, 1, 16384), _between(rng, 64, 8192 if dtype == "bf16" else 4096)
    return _pack(rng.choice(("restore", "backward")), rows, width, dtype,
                 rng.choice(("relu", "gelu", "sigmoid", "tanh")))


# ------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(std).add_(mean).to(kind)

    rows, width = case["rows"], case["width"]
    if case["op"] == "ce":
        vocab = case["vocab"]
        hidden, weight = normal(rows, width), normal(vocab, width, std=2.0 / math.sqrt(width))
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        if rows > 1:  # padding and prompt tokens carry no loss
            targets[torch.rand(rows, generator=gen, device="cuda") < 0.1] = -100
        counted = (targets >= 0).sum().clamp(min=1)
        grad_loss = torch.ones(rows, device="cuda") / counted
        return dict(case=case, hidden=hidden, weight=weight, targets=targets, grad_loss=grad_loss,
                    bias=normal(vocab, std=0.5) if case["bias"] else None)
    if case["op"] == "pack":
        spread = torch.randn(rows, width, generator=gen, device="cuda").mul_(0.5).exp_()
        x = (torch.randn(rows, width, generator=gen, device="cuda") * spread).to(kind)
        if case["call"] == "restore":
            return dict(case=case, x=x)
        codes, scales = _plain_pack(x.float())
        return dict(case=case, codes=codes.to(torch.int8), scales=scales, d_out=normal(rows, width))
    groups = case["groups"]
    state = dict(
        case=case, stream=normal(rows, width, std=2.0), branch=normal(rows, width, std=0.7),
        gate=normal(groups, width, std=0.3, mean=1.0) if groups else None,
        post_weight=normal(width, std=0.2, mean=1.0) if case["post"] else None,
        post_bias=normal(width, std=0.1) if case["post"] and case["bias"] else None,
        pre_weight=normal(width, std=0.2, mean=1.0), pre_bias=normal(width, std=0.1) if case["bias"] else None,
        stream_scale=1.0, branch_scale=0.5, eps=1e-6)
    if case["call"] == "backward":
        new, _, stats = _plain_norm(state)
        state.update(new_stream=new.to(kind), stats=stats, d_normed=normal(rows, width), d_stream=normal(rows, width))
        del state["stream"]
    return state


# ------------------------------------------------------------------------------ plain forms
def _plain_loss(s):
    hidden, valid = s["hidden"].float(), (s["targets"] >= 0) & (s["targets"] < s["weight"].shape[0])
    hidden = torch.where(valid[:, None], hidden, 0.0)
    logits = hidden @ s["weight"].float().T
    if s["bias"] is not None:
        logits += s["bias"].float()
    top = logits.amax(1, keepdim=True)
    lse = (logits - top).exp_().sum(1).log() + top[:, 0]
    picked = logits.gather(1, s["targets"].clamp(0, logits.shape[1] - 1)[:, None])[:, 0]
    loss = torch.where(valid, lse - picked, 0.0)
    return hidden, logits, valid, torch.where(valid, lse, 0.0), loss


def _plain_ce(s):
    kind = s["weight"].dtype
    hidden, logits, valid, lse, loss = _plain_loss(s)
    out = dict(loss=loss, lse=lse)
    if s["case"]["call"] == "train":
        slope = logits.sub_(lse[:, None]).exp_()
        at = s["targets"].clamp(0, logits.shape[1] - 1)[:, None]
        slope.scatter_(1, at, slope.gather(1, at) - 1.0)
        slope *= torch.where(valid, s["grad_loss"], 0.0)[:, None]
        slope = torch.where(valid[:, None], slope, 0.0)
        out["d_hidden"] = (slope @ s["weight"].float()).to(kind)
        out["d_weight"] = (slope.T @ hidden).to(kind)
        if s["bias"] is not None:
            out["d_bias"] = slope.sum(0).to(kind)
    return out


def _statistics(v, kind, eps):
    mean = v.mean(1) if kind == "layer" else torch.zeros_like(v[:, 0])
    return mean, 1.0 / ((v - mean[:, None]).square().mean(1) + eps).sqrt()


def _gates(s, rows):
    """The gate of every row."""
    gate = s["gate"].float()
    return gate.repeat_interleave(rows // gate.shape[0], 0)


def _affine(v, weight, bias):
    v = v if weight is None else v * weight.float()
    return v if bias is None else v + bias.float()


def _plain_norm(s):
    """The new residual stream, its norm and the statistics, in 32 bits."""
    kind, v = s["case"]["kind"], s["branch"].float()
    zero = torch.zeros_like(v[:, 0])
    stats = [zero, zero]
    if s["case"]["post"]:
        stats = _statistics(v, kind, s["eps"])
        v = _affine((v - stats[0][:, None]) * stats[1][:, None], s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        v = v * _gates(s, v.shape[0])
    new = s["stream_scale"] * s["stream"].float() + s["branch_scale"] * v
    mean, rstd = _statistics(new, kind, s["eps"])
    normed = _affine((new - mean[:, None]) * rstd[:, None], s["pre_weight"], s["pre_bias"])
    return new, normed, torch.stack([*stats, mean, rstd], 1)


def _norm_slope(slope, normal, rstd, kind):
    """The gradient of a norm's input from that of its normalised values."""
    slope_mean = slope.mean(1, keepdim=True) if kind == "layer" else 0.0
    return rstd[:, None] * (slope - slope_mean - normal * (slope * normal).mean(1, keepdim=True))


def _plain_norm_backward(s):
    kind, to = s["case"]["kind"], s["branch"].dtype
    post_mean, post_rstd, pre_mean, pre_rstd = s["stats"].unbind(1)
    d_normed, rows = s["d_normed"].float(), s["branch"].shape[0]
    normal = (s["new_stream"].float() - pre_mean[:, None]) * pre_rstd[:, None]
    out = dict(d_pre_weight=(d_normed * normal).sum(0))
    if s["pre_bias"] is not None:
        out["d_pre_bias"] = d_normed.sum(0)
    new = s["d_stream"].float() + _norm_slope(d_normed * s["pre_weight"].float(), normal, pre_rstd, kind)
    out["d_stream"] = s["stream_scale"] * new
    value = s["branch"].float()
    if s["case"]["post"]:
        normal = (value - post_mean[:, None]) * post_rstd[:, None]
        value = _affine(normal, s["post_weight"], s["post_bias"])
    slope = s["branch_scale"] * new
    if s["gate"] is not None:
        groups = s["gate"].shape[0]
        out["d_gate"] = (slope * value).view(groups, rows // groups, -1).sum(1)
        slope = slope * _gates(s, rows)
    if s["case"]["post"]:
        out["d_post_weight"] = (slope * normal).sum(0)
        if s["post_bias"] is not None:
            out["d_post_bias"] = slope.sum(0)
        slope = _norm_slope(slope * s["post_weight"].float(), normal, post_rstd, kind)
    out["d_branch"] = slope
    return {name: v.to(to) for name, v in out.items()}


def _blocks(x):
    """[rows, blocks, BLOCK], the last block filled up with zeros."""
    rows, width = x.shape
    count = -(-width // BLOCK)
    return torch.nn.functional.pad(x, (0, count * BLOCK - width)).view(rows, count, BLOCK)


def _plain_pack(x):
    """Codes (whole numbers in 32 bits) and scales of a matrix in 32 bits."""
    blocks = _blocks(x)
    most = blocks.abs().amax(2)
    full = torch.full_like(most, 127.0)
    some = most >= TINY
    codes = torch.where(some[:, :, None], (blocks * (full / most)[:, :, None]).round(), 0.0)
    return codes.view(x.shape[0], -1)[:, :x.shape[1]].contiguous(), torch.where(some, most / full, 0.0)


def _plain_unpack(codes, scales):
    return (_blocks(codes.float()) * scales[:, :, None]).view(codes.shape[0], -1)[:, :codes.shape[1]]


def _function(x, act, slope=False):
    """f(x), or f'(x)."""
    if act == "relu":
        return (x > 0).to(x.dtype) if slope else torch.where(x > 0, x, 0.0)
    if act == "sigmoid":
        y = 1.0 / (1.0 + (-x).exp())
        return y * (1.0 - y) if slope else y
    root = math.sqrt(2.0 / math.pi)
    t = (x if act == "tanh" else root * (x + 0.044715 * x * x * x)).tanh()
    if act == "tanh":
        return 1.0 - t * t if slope else t
    if not slope:
        return 0.5 * x * (1.0 + t)
    return 0.5 * (1.0 + t) + 0.5 * x * root * (1.0 + 3 * 0.044715 * x * x) * (1.0 - t * t)


def _plain_pack_case(s):
    act = s["case"]["act"]
    if s["case"]["call"] == "restore":
        x = s["x"].float()
        values = _plain_unpack(*_plain_pack(x))
        return dict(out=_function(x, act).to(s["x"].dtype), values=values.to(s["x"].dtype))
    x, kind = _plain_unpack(s["codes"], s["scales"]), s["d_out"].dtype
    return dict(d_preact=(s["d_out"].float() * _function(x, act, True)).to(kind), out=_function(x, act).to(kind))


# ------------------------------------------------------------------------------ the framework's calls
def _own(s):
    import deepity_b200 as dp

    case = s["case"]
    if case["op"] == "ce":
        args = s["hidden"], s["weight"], s["targets"]
        loss, lse = dp.vocab_cross_entropy(*args, s["bias"])
        out = dict(loss=loss, lse=lse)
        if case["call"] == "train":
            grads = dp.vocab_cross_entropy_backward(s["grad_loss"], *args, lse, s["bias"])
            out.update(d_hidden=grads.hidden, d_weight=grads.weight)
            if s["bias"] is not None:
                out["d_bias"] = grads.bias
        return out
    if case["op"] == "pack":
        if case["call"] == "restore":
            out, packed = dp.activate_and_pack(s["x"], case["act"])
            return dict(out=out, values=packed.unpack(s["x"].dtype))
        packed = dp.PackedActivations(s["codes"], s["scales"])
        d_preact, out = dp.packed_activation_backward(s["d_out"], packed, case["act"], recompute=True)
        return dict(d_preact=d_preact, out=out)
    block = {k: s[k] for k in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias", "stream_scale",
                               "branch_scale")}
    block.update(norm=case["kind"], post_norm=case["post"])
    if case["call"] == "forward":
        new, normed, stats = dp.residual_norm(s["stream"], s["branch"], eps=s["eps"], **block)
        return dict(new_stream=new, normed=normed, stats=stats)
    grads = dp.residual_norm_backward(s["d_normed"], s["d_stream"], s["new_stream"], s["branch"], s["stats"], **block)
    found = dict(d_pre_weight=grads.pre_weight, d_pre_bias=grads.pre_bias, d_stream=grads.stream, d_gate=grads.gate,
                 d_post_weight=grads.post_weight, d_post_bias=grads.post_bias, d_branch=grads.branch)
    return {name: v for name, v in found.items() if v is not None}


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "ce":
        return _plain_ce(state)
    if case["op"] == "pack":
        return _plain_pack_case(state)
    if case["call"] == "backward":
        return _plain_norm_backward(state)
    new, normed, stats = _plain_norm(state)
    kind = state["branch"].dtype
    return dict(new_stream=new.to(kind), normed=normed.to(kind), stats=stats)


# ------------------------------------------------------------------------------ what a pass needs
def work(case):
    size, rows, width = TYPES[case["dtype"]].itemsize, case["rows"], case["width"]
    cells, train = rows * width, case["call"] in ("train", "backward")
    if case["op"] == "ce":
        params = case["vocab"] * (width + case["bias"])
        return {"bytes": (cells + params) * size * (2 if train else 1) + rows * (20 if train else 16),
                "flops": (6 if train else 2) * cells * case["vocab"]}
    if case["op"] == "pack":
        kept = cells + 4 * rows * -(-width // BLOCK)
        return {"bytes": 3 * cells * size + (kept if train else 0), "flops": 10 * cells}
    gate = case["groups"] * width
    vectors = gate + width * (1 + case["post"]) * (1 + case["bias"])
    if train:
        return {"bytes": (6 * cells + 2 * vectors) * size + 16 * rows, "flops": 30 * cells}
    return {"bytes": (4 * cells + vectors) * size + 16 * rows, "flops": 15 * cells}


# ------------------------------------------------------------------------------ in 64 bits
def _exact_ce(case, s):
    hidden, weight, targets = s["hidden"].double(), s["weight"].double(), s["targets"]
    bias = s["bias"].double() if s["bias"] is not None else torch.zeros(weight.shape[0], device="cuda").double()
    kept = ((targets >= 0) & (targets < len(weight))).nonzero()[:, 0]
    loss, lse = torch.zeros(len(hidden), device="cuda").double(), torch.zeros(len(hidden), device="cuda").double()
    d_hidden, d_weight, d_bias = torch.zeros_like(hidden), torch.zeros_like(weight), torch.zeros_like(bias)
    for some in kept.split(2048):
        logits = torch.addmm(bias, hidden[some], weight.T)
        lse[some] = torch.logsumexp(logits, 1)
        loss[some] = torch.nn.functional.cross_entropy(logits, targets[some], reduction="none")
        if case["call"] == "train":
            slope = torch.softmax(logits, 1)
            slope[torch.arange(len(some), device="cuda"), targets[some]] -= 1
            slope *= s["grad_loss"][some].double()[:, None]
            d_hidden[some] = slope @ weight
            d_weight.addmm_(slope.T, hidden[some])
            d_bias += slope.sum(0)
    out = dict(loss=loss, lse=lse)
    if case["call"] == "train":
        out.update(d_hidden=d_hidden, d_weight=d_weight)
        if case["bias"]:
            out["d_bias"] = d_bias
    return out


def _exact_norm(case, s):
    """The forward pass in 64 bits; its gradients by differentiation, from the stream that was kept."""
    def norm(v, weight, bias, mean=None, rstd=None):
        if rstd is None:
            mean = v.mean(1, keepdim=True) if case["kind"] == "layer" else 0.0
            rstd = torch.rsqrt(((v - mean) ** 2).mean(1, keepdim=True) + s["eps"])
        v = (v - mean) * rstd
        v = v if weight is None else v * weight
        return (v if bias is None else v + bias), mean, rstd

    wide = {k: v.double() if torch.is_tensor(v) else v for k, v in s.items()}
    rows, zero = case["rows"], torch.zeros(case["rows"], 1, device="cuda").double()
    gate = wide["gate"]
    if case["call"] == "forward":
        u, mean, rstd = wide["branch"], zero, zero
        if case["post"]:
            u, mean, rstd = norm(u, wide["post_weight"], wide["post_bias"])
        if gate is not None:
            u = (u.view(len(gate), -1, case["width"]) * gate[:, None]).view(u.shape)
        new = s["stream_scale"] * wide["stream"] + s["branch_scale"] * u
        normed, mean2, rstd2 = norm(new, wide["pre_weight"], wide["pre_bias"])
        stats = [m + zero for m in (mean, rstd, mean2, rstd2)]
        return dict(new_stream=new, normed=normed, stats=torch.cat(stats, 1))

    # A norm's gradient is linear in its output's: J^T d, with J of v -> (v - mean) * rstd written out.
    def pull(d, v, mean, rstd):
        n = (v - mean) * rstd
        back = d - n * ((d * n).sum(1, keepdim=True) / v.shape[1])
        if case["kind"] == "layer":
            back = back - d.sum(1, keepdim=True) / v.shape[1]
        return back * rstd, n

    m1, r1, m2, r2 = wide["stats"].split(1, 1)
    d_new, n2 = pull(wide["d_normed"] * wide["pre_weight"], wide["new_stream"], m2, r2)
    d_new = d_new + wide["d_stream"]
    out = dict(d_pre_weight=torch.einsum("rw,rw->w", wide["d_normed"], n2))
    if case["bias"]:
        out["d_pre_bias"] = wide["d_normed"].sum(0)
    out["d_stream"] = d_new * s["stream_scale"]
    u = norm(wide["branch"], wide["post_weight"], wide["post_bias"], m1, r1)[0] if case["post"] else wide["branch"]
    d_u = d_new * s["branch_scale"]
    if gate is not None:
        parts = (len(gate), rows // len(gate), case["width"])
        out["d_gate"] = torch.einsum("grw,grw->gw", d_u.view(parts), u.view(parts))
        d_u = (d_u.view(parts) * gate[:, None]).view(rows, -1)
    if case["post"]:
        d_branch, n1 = pull(d_u * wide["post_weight"], wide["branch"], m1, r1)
        out["d_post_weight"] = torch.einsum("rw,rw->w", d_u, n1)
        if case["bias"]:
            out["d_post_bias"] = d_u.sum(0)
        d_u = d_branch
    out["d_branch"] = d_u
    return out


def _exact_pack(case, s):
    functions = {"relu": torch.relu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
                 "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}
    f, width = functions[case["act"]], case["width"]
    if case["call"] == "restore":
        x, values = s["x"].double(), torch.zeros_like(s["x"]).double()
        for at in range(0, width, BLOCK):
            part = x[:, at:at + BLOCK]
            step = part.abs().amax(1, keepdim=True) / 127
            some = step >= TINY / 127
            values[:, at:at + BLOCK] = torch.where(some, torch.round(part / step) * step, 0.0)
        return dict(out=f(x), values=values)
    scales = s["scales"].double().repeat_interleave(BLOCK, 1)[:, :width]
    x = (s["codes"].double() * scales).requires_grad_()
    y = f(x)
    slope, = torch.autograd.grad(y, x, s["d_out"].double())
    return dict(d_preact=slope, out=y.detach())


def exact(case, seed):
    s = prepare(case, seed)
    return {"ce": _exact_ce, "norm": _exact_norm, "pack": _exact_pack}[case["op"]](case, s)
