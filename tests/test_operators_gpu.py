"""The operators of deepity_b200/operators.py on the GPU against 64-bit references (tests/operators_common.py, where the
tolerances are derived): the loss over a large vocabulary, the residual norms, packed activations, and a
training step of a small residual stack through all of them."""
import ctypes

import pytest
import torch

import operators_common as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dp(built_library):
    import deepity_b200
    return deepity_b200


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)


# ------------------------------------------------------------------------------ vocabulary loss
def vocab_case(rows, width, vocab, kind, bias=False, seed=0, ignore=0.15):
    g = gen(seed)
    hidden = normal(g, rows, width, dtype=kind)
    weight = normal(g, vocab, width, dtype=kind, std=2.0 / width ** 0.5)
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if rows > 2:
        targets[torch.rand(rows, generator=g, device="cuda") < ignore] = -100
    b = normal(g, vocab, dtype=kind) if bias else None
    return hidden, weight, targets, b


def check_vocab(dp, hidden, weight, targets, bias=None, scale=1.0, ignore_index=-100, grad=None):
    rows = targets.numel()
    if grad is None:
        grad = torch.linspace(0.5, 2.0, rows, device="cuda").view(targets.shape) / max(1, rows)
    want = ref.vocab_reference(hidden.reshape(rows, -1), weight, targets.reshape(-1), bias, scale, ignore_index,
                               grad.reshape(-1))
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias, scale=scale, ignore_index=ignore_index)
    ref.check(loss.reshape(-1), want["loss"], "loss")
    ref.check(lse.reshape(-1), want["lse"], "lse")
    got = dp.vocab_cross_entropy_backward(grad, hidden, weight, targets, lse, bias, scale=scale, ignore_index=ignore_index)
    ref.check(got.hidden.reshape(rows, -1), want["hidden"], "d_hidden")
    ref.check(got.weight, want["weight"], "d_weight")
    if bias is None:
        assert got.bias is None
    else:
        ref.check(got.bias, want["bias"], "d_bias")
    return loss, lse, got


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,vocab", [
    (1, 64, 1), (1, 8, 300), (3, 1, 5), (2, 1024, 4099), (127, 96, 257), (128, 64, 256), (129, 65, 255),
    (257, 72, 1000), (300, 515, 777), (513, 256, 2053), (33, 2048, 600),
    (4, 512, 3001), (5, 1000, 1111), (8, 513, 2222), (9, 264, 700)])
def test_vocab_sizes(dp, rows, width, vocab, kind):
    check_vocab(dp, *vocab_case(rows, width, vocab, TYPES[kind], seed=rows + width))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_vocab_bias_scale_and_ignored_index(dp, kind):
    hidden, weight, targets, bias = vocab_case(200, 120, 1003, TYPES[kind], bias=True, seed=3)
    targets[5], targets[9], targets[11] = 1003, -1, 1 << 40  # outside: ignored like -100
    check_vocab(dp, hidden, weight, targets, bias, scale=0.25)
    targets[::3] = 7
    loss, lse, got = check_vocab(dp, hidden, weight, targets, bias, ignore_index=7)
    assert not loss[::3].any() and not lse[::3].any() and not got.hidden[::3].any()


def test_vocab_one_gradient_for_all_rows(dp):
    hidden, weight, targets, _ = vocab_case(70, 64, 500, torch.bfloat16, seed=4)
    loss, lse, each = check_vocab(dp, hidden, weight, targets, grad=torch.full((70,), 0.125, device="cuda"))
    for one in (torch.tensor(0.125, device="cuda"), torch.tensor([0.125], device="cuda"),
                torch.tensor(0.125, device="cuda").expand(70)):
        got = dp.vocab_cross_entropy_backward(one, hidden, weight, targets, lse)
        assert torch.equal(got.hidden, each.hidden) and torch.equal(got.weight, each.weight)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_vocab_ignored_rows_may_hold_anything(dp, kind):
    hidden, weight, targets, bias = vocab_case(150, 88, 640, TYPES[kind], bias=True, seed=5)
    targets[3], targets[77], targets[149] = -100, -100, 640
    grad = torch.rand(150, generator=gen(1), device="cuda")
    clean = check_vocab(dp, hidden, weight, targets, bias, grad=grad)
    dirty, dirty_grad = hidden.clone(), grad.clone()
    dirty[3], dirty[77, 5], dirty[149] = float("nan"), float("inf"), -float("inf")
    dirty_grad[3], dirty_grad[77], dirty_grad[149] = float("nan"), float("inf"), 1e38
    loss, lse = dp.vocab_cross_entropy(dirty, weight, targets, bias)
    got = dp.vocab_cross_entropy_backward(dirty_grad, dirty, weight, targets, lse, bias)
    assert torch.equal(loss, clean[0]) and torch.equal(lse, clean[1])
    for a, b in zip(got, clean[2]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_vocab_nothing_counts(dp, kind):
    hidden, weight, targets, bias = vocab_case(40, 32, 300, TYPES[kind], bias=True, seed=6)
    targets.fill_(-100)
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    got = dp.vocab_cross_entropy_backward(torch.ones(40, device="cuda"), hidden, weight, targets, lse, bias)
    for t in (loss, lse, *got):
        assert not t.any()


def test_vocab_masked_words(dp):
    """A bias of -inf takes a word out; a masked target has an infinite loss; one word left has loss 0."""
    hidden, weight, targets, bias = vocab_case(64, 40, 700, torch.float32, bias=True, seed=7, ignore=0.0)
    bias[300:620] = -float("inf")
    targets[:] = torch.randint(0, 300, (64,), generator=gen(2), device="cuda")
    check_vocab(dp, hidden, weight, targets, bias)
    targets[0] = 400
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    assert loss[0] == float("inf") and lse.isfinite().all() and loss[1:].isfinite().all()
    bias[:], bias[650] = -float("inf"), 1.0
    targets[:] = 650
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    assert not loss.any()


def test_vocab_lowest_bias(dp):
    hidden, weight, targets, bias = vocab_case(32, 24, 400, torch.float32, bias=True, seed=8, ignore=0.0)
    bias[200:] = torch.finfo(torch.float32).min / 2
    targets %= 200
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    less = dp.vocab_cross_entropy(hidden, weight[:200], targets, bias[:200])
    assert torch.equal(loss, less[0]) and torch.equal(lse, less[1])


def test_vocab_nan_in_a_counted_row_stays_in_its_row(dp):
    hidden, weight, targets, _ = vocab_case(140, 64, 512, torch.bfloat16, seed=9, ignore=0.0)
    clean = dp.vocab_cross_entropy(hidden, weight, targets)
    hidden[131, 7] = float("nan")
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets)
    assert loss[131].isnan() and lse[131].isnan()
    keep = torch.arange(140, device="cuda") != 131
    assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(lse[keep], clean[1][keep])


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("left,pad", [(0, 8), (8, 16), (1, 3), (3, 13)])
def test_vocab_strides_and_alignment(dp, kind, left, pad):
    hidden, weight, targets, _ = vocab_case(90, 64, 333, TYPES[kind], seed=10)
    wide_h = torch.full((90, 64 + pad), float("nan"), device="cuda", dtype=TYPES[kind])
    wide_w = torch.full((333, 64 + pad), float("nan"), device="cuda", dtype=TYPES[kind])
    h, w = wide_h[:, min(left, pad):][:, :64], wide_w[:, min(left, pad):][:, :64]
    h.copy_(hidden), w.copy_(weight)
    want = check_vocab(dp, hidden, weight, targets)
    got = check_vocab(dp, h, w, targets)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2].weight, want[2].weight)


def test_vocab_leading_dimensions(dp):
    hidden, weight, targets, _ = vocab_case(60, 64, 333, torch.bfloat16, seed=11)
    flat = check_vocab(dp, hidden, weight, targets)
    loss, lse, got = check_vocab(dp, hidden.view(3, 4, 5, 64), weight, targets.view(3, 4, 5))
    assert loss.shape == (3, 4, 5) and got.hidden.shape == (3, 4, 5, 64)
    assert torch.equal(loss.view(-1), flat[0]) and torch.equal(got.hidden.view(60, 64), flat[2].hidden)


@pytest.mark.parametrize("rows,width,vocab,kind", [(16384, 64, 20000, "bf16"), (6000, 40, 9000, "f32"),
                                                   (5, 2048, 30000, "f32")])
def test_vocab_pieces(dp, rows, width, vocab, kind):
    """More than one piece of the vocabulary, in the gradient or in the copies of the weights."""
    check_vocab(dp, *vocab_case(rows, width, vocab, TYPES[kind], bias=True, seed=12))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9])
def test_vocab_few_rows_with_bias_and_ignored_ones(dp, rows, kind):
    hidden, weight, targets, bias = vocab_case(rows, 200, 2500, TYPES[kind], bias=True, seed=30 + rows, ignore=0.0)
    check_vocab(dp, hidden, weight, targets, bias, scale=0.5)
    want = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    targets[-1] = -100
    hidden[-1] = float("nan")
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    assert torch.equal(loss[:-1], want[0][:-1]) and torch.equal(lse[:-1], want[1][:-1])
    assert loss[-1] == 0 and lse[-1] == 0


@pytest.mark.parametrize("rows", [1, 2, 40])
def test_vocab_every_word_masked(dp, rows):
    """The sum of no exponentials: its logarithm is -inf, the loss no number; ignored rows stay 0."""
    hidden, weight, targets, bias = vocab_case(rows, 32, 300, torch.float32, bias=True, seed=31, ignore=0.0)
    bias.fill_(-float("inf"))
    if rows > 1:
        targets[1] = -100
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    counted = targets >= 0
    assert (lse[counted] == -float("inf")).all() and loss[counted].isnan().all()
    assert not loss[~counted].any() and not lse[~counted].any()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [2, 30])
def test_vocab_large_logits(dp, rows, kind):
    """Logits of some thousands: exponentials of differences only."""
    hidden, weight, targets, _ = vocab_case(rows, 64, 600, TYPES[kind], seed=32, ignore=0.0)
    check_vocab(dp, hidden, weight, targets, scale=1000.0)


def test_vocab_unequal_gradients(dp):
    """Gradients of the losses over many orders of magnitude, zeros and signs among them."""
    hidden, weight, targets, bias = vocab_case(64, 48, 500, torch.float32, bias=True, seed=33)
    grad = 10.0 ** torch.linspace(-20, 3, 64, device="cuda") * torch.where(torch.arange(64, device="cuda") % 3 == 0, -1.0, 1.0)
    grad[10:14] = 0.0
    check_vocab(dp, hidden, weight, targets, bias, grad=grad)
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    got = dp.vocab_cross_entropy_backward(torch.zeros(64, device="cuda"), hidden, weight, targets, lse, bias)
    assert not got.hidden.any() and not got.weight.any() and not got.bias.any()


def test_vocab_offsets_beyond_32_bits(dp):
    """A weight of 2^32 elements and more: the last words are read and written where they are."""
    width, vocab = 8192, (1 << 19) + 65
    weight = torch.zeros(vocab, width, device="cuda", dtype=torch.bfloat16)
    g = gen(34)
    weight[-40:] = normal(g, 40, width, dtype=torch.bfloat16, std=0.05)
    hidden = normal(g, 3, width, dtype=torch.bfloat16)
    targets = torch.tensor([vocab - 1, vocab - 30, 5], device="cuda")
    logits = hidden.double() @ weight[-40:].double().T
    lse = torch.logsumexp(torch.cat([logits, torch.full((3, 1), float(vocab - 40), device="cuda").double().log()], 1), 1)
    loss, found = dp.vocab_cross_entropy(hidden, weight, targets)
    picked = torch.stack([logits[0, 39], logits[1, 10], torch.zeros((), device="cuda").double()])
    assert (found.double() - lse).abs().max() < 1e-3 and (loss.double() - (lse - picked)).abs().max() < 1e-3
    got = dp.vocab_cross_entropy_backward(torch.ones(3, device="cuda"), hidden, weight, targets, found)
    slope = torch.exp(logits - lse[:, None])
    slope[0, 39] -= 1
    slope[1, 10] -= 1
    want = slope.T @ hidden.double()
    # s and the result rounded to bf16, half a step each, and 1e-3 of lse's error in every probability
    bound = (2 * 2.0 ** -8 + 2e-3) * (slope.abs().T @ hidden.double().abs()) + 2.0 ** -8 * want.abs()
    assert ((got.weight[-40:].double() - want).abs() <= bound).all()
    assert (got.weight[5].double() + hidden[2].double()).abs().max() < 2.0 ** -7 * hidden[2].double().abs().max()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_vocab_no_rows(dp, kind):
    hidden = torch.empty(0, 16, device="cuda", dtype=TYPES[kind])
    weight = normal(gen(0), 30, 16, dtype=TYPES[kind])
    targets = torch.empty(0, device="cuda", dtype=torch.int64)
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, weight[:, 0].contiguous())
    assert loss.shape == (0,)
    got = dp.vocab_cross_entropy_backward(loss, hidden, weight, targets, lse, weight[:, 0].contiguous())
    assert got.hidden.shape == (0, 16) and not got.weight.any() and not got.bias.any()


def test_vocab_gradient_against_differences(dp):
    hidden, weight, targets, bias = vocab_case(20, 12, 90, torch.float32, bias=True, seed=13)
    total = lambda *a: dp.vocab_cross_entropy(*a)[0].double().sum()  # noqa: E731
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    got = dp.vocab_cross_entropy_backward(torch.ones(20, device="cuda"), hidden, weight, targets, lse, bias)
    g = gen(14)
    for at, slope in ((0, got.hidden), (1, got.weight), (3, got.bias)):
        args = [hidden, weight, targets, bias]
        step = normal(g, *args[at].shape)
        want = (slope.double() * step).sum()
        # central differences: third derivatives of a sum of 20 losses along a unit-sized step are below 100 in
        # these units, so h = 2^-7 leaves 100 h^2 / 6 = 1e-3; the losses' own 1e-6 each leave 20e-6 / h = 2.6e-3
        h = 2.0 ** -7
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[at] = args[at] + sign * h * step
            ends.append(total(*moved))
        assert abs((ends[0] - ends[1]) / (2 * h) - want) < 0.01 * max(1.0, abs(float(want)))


def _c_vocab(dp, hidden, weight, targets, **more):
    from deepity_b200 import _lib
    rows, width = hidden.shape
    return _lib.VocabCe(rows=rows, width=width, vocab=weight.shape[0], hidden_stride=hidden.stride(0),
                        weight_stride=weight.stride(0), type=0 if hidden.dtype == torch.float32 else 1, scale=1.0,
                        ignore_index=-100, hidden=hidden.data_ptr(), weight=weight.data_ptr(),
                        targets=targets.data_ptr(), **more)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("pad", [5, 8])
def test_vocab_c_entry_writes_its_own_elements_only(dp, kind, pad):
    """Gradients into rows with gaps: what lies in the gaps and behind the last row stays."""
    from deepity_b200 import _lib
    lib, kind = _lib.load(), TYPES[kind]
    hidden, weight, targets, _ = vocab_case(131, 72, 301, kind, seed=15)
    loss, lse, want = check_vocab(dp, hidden, weight, targets, grad=torch.ones(131, device="cuda"))
    d_hidden = torch.full((133, 72 + pad), 7.0, device="cuda", dtype=kind)
    d_weight = torch.full((303, 72 + pad), 7.0, device="cuda", dtype=kind)
    one = torch.ones(1, device="cuda")
    c = _c_vocab(dp, hidden, weight, targets, lse=lse.data_ptr(), grad_loss=one.data_ptr(), grad_stride=0,
                 d_hidden=d_hidden.data_ptr(), d_weight=d_weight.data_ptr(), d_hidden_stride=72 + pad,
                 d_weight_stride=72 + pad)
    size = ctypes.c_size_t()
    _lib.check(lib.dpc_vocab_ce_workspace(ctypes.byref(c), 1, ctypes.byref(size)))
    ws = torch.full((size.value + 256,), 0xAB, device="cuda", dtype=torch.uint8)  # (dirty, and watched behind its end)
    c.workspace, c.workspace_bytes = ws.data_ptr(), size.value
    _lib.check(lib.dpc_vocab_ce_backward(torch.cuda.current_stream().cuda_stream, ctypes.byref(c)))
    assert torch.equal(d_hidden[:131, :72], want.hidden) and torch.equal(d_weight[:301, :72], want.weight)
    assert (d_hidden[:, 72:] == 7).all() and (d_hidden[131:] == 7).all()
    assert (d_weight[:, 72:] == 7).all() and (d_weight[301:] == 7).all()
    assert (ws[size.value:] == 0xAB).all()
    c.workspace_bytes -= 1
    assert lib.dpc_vocab_ce_backward(None, ctypes.byref(c)) == -1 and b"workspace" in lib.dpc_last_error()


# ------------------------------------------------------------------------------ residual norms
def norm_case(rows, width, kind, gate=None, post=True, bias=False, branch=True, seed=0, mean=0.0):
    g = gen(seed)
    c = dict(stream=normal(g, rows, width, dtype=kind, std=2.0, mean=mean),
             branch=normal(g, rows, width, dtype=kind, std=0.7, mean=mean) if branch else None,
             gate=None if gate is None else normal(g, *gate, dtype=kind, std=0.4, mean=1.0),
             post_weight=normal(g, width, dtype=kind, std=0.2, mean=1.0) if post else None,
             post_bias=normal(g, width, dtype=kind, std=0.1) if post and bias else None,
             pre_weight=normal(g, width, dtype=kind, std=0.2, mean=1.0),
             pre_bias=normal(g, width, dtype=kind, std=0.1) if bias else None)
    return c, normal(g, rows, width, dtype=kind), normal(g, rows, width, dtype=kind)


def check_norm(dp, c, d_normed, d_stream, norm, a=1.0, b=1.0, eps=1e-5, post_norm=None):
    c = dict(c)
    stream, branch = c.pop("stream"), c.pop("branch")
    post = c["post_weight"] is not None if post_norm is None else post_norm
    new, normed, stats = dp.residual_norm(stream, branch, norm=norm, post_norm=post_norm, stream_scale=a,
                                          branch_scale=b, eps=eps, **c)
    want = ref.norm_reference(stream, branch, norm, post, c["post_weight"], c["post_bias"], c["gate"], a, b,
                              c["pre_weight"], c["pre_bias"], eps)
    if branch is None:
        assert new is stream
    else:
        ref.check(new, want["new"], "new_stream")
    ref.check(normed, want["normed"], "normed")
    ref.check(stats, want["stats"], "stats")
    got = dp.residual_norm_backward(d_normed, d_stream, new, branch, stats, norm=norm, post_norm=post_norm,
                                    stream_scale=a, branch_scale=b, **c)
    want = ref.norm_backward_reference(d_normed, d_stream, new, branch, stats, norm, post, c["post_weight"],
                                       c["post_bias"], c["gate"], a, b, c["pre_weight"], c["pre_bias"])
    given = dict(c, stream=stream, branch=branch)
    for name, value in got._asdict().items():
        if given[name] is None:
            assert value is None, name
        else:
            assert value.dtype == stream.dtype
            ref.check(value, want[name], "d_" + name)
    return new, normed, stats, got


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 64), (7, 3), (5, 512), (64, 513), (33, 1023), (130, 2048),
                                        (9, 2056), (40, 4096), (3, 4097), (6, 8192), (5, 8200), (4, 16384), (2, 12345)])
def test_norm_sizes(dp, rows, width, norm, kind):
    c, d_normed, d_stream = norm_case(rows, width, TYPES[kind], gate=(width,), bias=True, seed=rows)
    check_norm(dp, c, d_normed, d_stream, norm, a=0.9, b=0.5)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("gate,post,bias,branch,stream", [
    (None, True, False, True, True), (None, False, False, True, True), ((4, 136), True, True, True, True),
    ((1, 136), False, False, True, False), ((60, 136), True, False, True, True), ((3, 4, 136), False, True, True, True),
    (None, False, True, False, True), (None, False, False, False, False)])
def test_norm_forms(dp, gate, post, bias, branch, stream, kind):
    for norm in ("rms", "layer"):
        c, d_normed, d_stream = norm_case(60, 136, TYPES[kind], gate, post, bias, branch, seed=2)
        check_norm(dp, c, d_normed, d_stream if stream else None, norm, a=0.8 if branch else 1.0, b=1.5)


def test_norm_without_weights(dp):
    c, d_normed, d_stream = norm_case(20, 300, torch.float32, post=False, seed=3)
    c["pre_weight"] = None
    for norm in ("rms", "layer"):
        check_norm(dp, c, d_normed, d_stream, norm, post_norm=True)


@pytest.mark.parametrize("rows,groups,width", [(5000, 1, 256), (5000, 2, 256), (4096, 1024, 64), (2222, 2222, 72),
                                               (3003, 3, 2048)])
def test_norm_many_rows(dp, rows, groups, width):
    c, d_normed, d_stream = norm_case(rows, width, torch.bfloat16, (groups, width), bias=True, seed=4)
    check_norm(dp, c, d_normed, d_stream, "rms", b=0.5)


def test_norm_large_mean(dp):
    """A mean a thousand times the deviation: the squares are taken of what is left of it."""
    c, d_normed, d_stream = norm_case(30, 640, torch.float32, bias=True, seed=5, mean=1000.0)
    check_norm(dp, c, d_normed, d_stream, "layer")


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("left,pad", [(0, 8), (1, 5), (8, 8)])
def test_norm_strides(dp, kind, left, pad):
    kind = TYPES[kind]
    c, d_normed, d_stream = norm_case(50, 128, kind, (5, 128), bias=True, seed=6)
    want = check_norm(dp, c, d_normed, d_stream, "layer")

    def spread(t):
        wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), device="cuda", dtype=kind)
        view = wide[:, min(left, pad):][:, :t.shape[1]]
        view.copy_(t)
        return view

    moved = dict(c, stream=spread(c["stream"]), branch=spread(c["branch"]), gate=spread(c["gate"]))
    check_norm(dp, moved, spread(d_normed), spread(d_stream), "layer")
    assert want[0].shape == (50, 128)


def test_norm_leading_dimensions_and_broadcast_gate(dp):
    c, d_normed, d_stream = norm_case(24, 64, torch.bfloat16, (4, 64), seed=7)
    flat = check_norm(dp, c, d_normed, d_stream, "rms")
    new, normed, stats = dp.residual_norm(c["stream"].view(4, 6, 64), c["branch"].view(4, 6, 64), gate=c["gate"],
                                          post_weight=c["post_weight"], pre_weight=c["pre_weight"], eps=1e-5)
    assert new.shape == (4, 6, 64) and stats.shape == (4, 6, 4)
    assert torch.equal(new.view(24, 64), flat[0]) and torch.equal(normed.view(24, 64), flat[1])


def test_norm_rows_of_zeros_and_of_nan(dp):
    c, d_normed, d_stream = norm_case(12, 96, torch.float32, seed=8)
    c["stream"][3], c["branch"][3] = 0.0, 0.0
    new, normed, stats, got = check_norm(dp, c, d_normed, d_stream, "rms")
    assert not new[3].any() and not normed[3].any()
    c["stream"][5, 1] = float("nan")
    dirty = dp.residual_norm(c["stream"], c["branch"], post_weight=c["post_weight"], pre_weight=c["pre_weight"], eps=1e-5)
    keep = torch.arange(12, device="cuda") != 5
    assert dirty[1][5].isnan().all() and torch.equal(dirty[1][keep], normed[keep])


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_norm_no_rows(dp, kind):
    kind = TYPES[kind]
    c, d_normed, d_stream = norm_case(4, 40, kind, (2, 40), bias=True, seed=9)
    empty = torch.empty(0, 40, device="cuda", dtype=kind)
    c["stream"], c["branch"] = empty, empty
    new, normed, stats = dp.residual_norm(**c)
    assert new.shape == normed.shape == (0, 40) and stats.shape == (0, 4)
    stream = c.pop("stream"), c.pop("branch")
    got = dp.residual_norm_backward(empty, empty, *stream, stats, **c)
    assert got.stream.shape == got.branch.shape == (0, 40)
    for t in (got.gate, got.post_weight, got.post_bias, got.pre_weight, got.pre_bias):
        assert t.numel() and not t.any()


def test_norm_gradient_against_differences(dp):
    c, d_normed, d_stream = norm_case(6, 40, torch.float32, (2, 40), bias=True, seed=10)
    for norm in ("rms", "layer"):
        def total(**given):
            new, normed, _ = dp.residual_norm(norm=norm, stream_scale=0.9, branch_scale=0.5, eps=1e-5, **given)
            return (new.double() * d_stream.double()).sum() + (normed.double() * d_normed.double()).sum()

        rest = {k: v for k, v in c.items() if k not in ("stream", "branch")}
        new, _, stats = dp.residual_norm(norm=norm, stream_scale=0.9, branch_scale=0.5, eps=1e-5, **c)
        got = dp.residual_norm_backward(d_normed, d_stream, new, c["branch"], stats, norm=norm, stream_scale=0.9,
                                        branch_scale=0.5, **rest)
        for name, slope in got._asdict().items():
            step = normal(gen(11), *c[name].shape)
            want = float((slope.double() * step).sum())
            # 240 elements of about 1, third derivatives of a norm below 10 each: h^2 / 6 * 2400 = 1.0 * h * h * 400;
            # roundings of 480 terms of 2^-22 each over 2h: 1e-4 / h at most
            h = 2.0 ** -8
            ends = [total(**{**c, name: c[name] + sign * h * step}) for sign in (1, -1)]
            assert abs(float(ends[0] - ends[1]) / (2 * h) - want) < 400 * h * h + 1e-4 / h, (norm, name)


def test_norm_and_pack_offsets_beyond_32_bits(dp):
    """Matrices of more than 2^32 elements: the last row is computed from and written to its place."""
    rows, width = (1 << 18) + 3, 16384
    x = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
    x[-1] = normal(gen(40), width, dtype=torch.bfloat16)
    weight = torch.ones(width, device="cuda", dtype=torch.bfloat16)
    few = dp.residual_norm(x[-1:].clone(), pre_weight=weight)
    _, normed, stats = dp.residual_norm(x, pre_weight=weight)
    assert torch.equal(normed[-1:], few[1]) and torch.equal(stats[-1:], few[2]) and not normed[:-1:4099].any()
    got = dp.residual_norm_backward(normed, None, x, None, stats, pre_weight=weight)
    want = dp.residual_norm_backward(few[1], None, x[-1:].clone(), None, few[2], pre_weight=weight)
    assert torch.equal(got.stream[-1:], want.stream) and torch.equal(got.pre_weight, want.pre_weight)
    del normed, got
    out, packed = dp.activate_and_pack(x, "gelu")
    single = dp.activate_and_pack(x[-1:].clone(), "gelu")
    assert torch.equal(out[-1:], single[0]) and torch.equal(packed.codes[-1:], single[1].codes)
    assert torch.equal(packed.scales[-1:], single[1].scales)
    del out
    d_x, _ = dp.packed_activation_backward(x, packed, "gelu")
    assert torch.equal(d_x[-1:], dp.packed_activation_backward(x[-1:].clone(), single[1], "gelu")[0])


def test_results_carry_no_history(dp):
    t = {k: v.requires_grad_() if v.is_floating_point() else v for k, v in step_inputs(50).items()}
    for out in one_step(dp, t):
        assert not out.requires_grad


def test_norm_c_entry_leaves_gaps_and_unwanted_gradients(dp):
    from deepity_b200 import _lib
    lib = _lib.load()
    c, d_normed, d_stream = norm_case(37, 200, torch.bfloat16, seed=12)
    new, normed, stats, want = check_norm(dp, c, d_normed, d_stream, "rms")
    d_in = torch.full((39, 208), 7.0, device="cuda", dtype=torch.bfloat16)
    call = _lib.ResidualNorm(rows=37, width=200, groups=1, type=1, norm=0, post_norm=1, stream_scale=1.0,
                             branch_scale=1.0, eps=1e-5, branch=c["branch"].data_ptr(), branch_stride=200,
                             post_weight=c["post_weight"].data_ptr(), pre_weight=c["pre_weight"].data_ptr(),
                             new_stream=new.data_ptr(), new_stream_stride=200, stats=stats.data_ptr(),
                             d_normed=d_normed.data_ptr(), d_normed_stride=200, d_new_stream=d_stream.data_ptr(),
                             d_new_stream_stride=200, d_stream=d_in.data_ptr(), d_stream_stride=208)
    size = ctypes.c_size_t()
    _lib.check(lib.dpc_residual_norm_workspace(ctypes.byref(call), ctypes.byref(size)))
    ws = torch.full((size.value + 256,), 0xAB, device="cuda", dtype=torch.uint8)
    call.workspace, call.workspace_bytes = ws.data_ptr(), size.value
    _lib.check(lib.dpc_residual_norm_backward(torch.cuda.current_stream().cuda_stream, ctypes.byref(call)))
    assert torch.equal(d_in[:37, :200], want.stream) and (d_in[:, 200:] == 7).all() and (d_in[37:] == 7).all()
    assert (ws[size.value:] == 0xAB).all()


# ------------------------------------------------------------------------------ packed activations
ACTS = ["relu", "gelu", "sigmoid", "esigmoid", "tanh", "linear", "hard_tanh"]


def check_pack(dp, x, act, d_out):
    kind = x.dtype
    out, packed = dp.activate_and_pack(x, act)
    codes, scales = ref.pack_reference(x.reshape(-1, x.shape[-1]))
    assert torch.equal(packed.codes.cpu().view(codes.shape), codes)
    assert torch.equal(packed.scales.cpu().view(scales.shape).nan_to_num(-1.0), scales.nan_to_num(-1.0))
    f, _, d_f, _ = ref.activation_reference(act, x.double())
    ref.check(out, (f, d_f + ref.half(kind) * f.abs() + 2 * ref.U * f.abs()), "out")
    kept = ref.unpack_reference(codes, scales).to(x.device).view(x.shape)
    for to in (torch.float32, torch.bfloat16):
        ref.check(packed.unpack(to), (kept, (ref.half(to) + 2 * ref.U) * kept.abs()), "values")
    assert ((kept - x.double()).abs() <= kept.abs() * 4 * ref.U + x.double().abs().amax() / 254 * (1 + 1e-5)).all()
    d_x, again = dp.packed_activation_backward(d_out, packed, act, recompute=True)
    # the reference takes the kept value as float32 holds it: one product
    f, slope, d_f, d_s = ref.activation_reference(act, kept.float().double())
    g = d_out.double()
    ref.check(d_x, (g * slope, g.abs() * (d_s + (ref.half(kind) + 16 * ref.U) * slope.abs())), "d_preact")
    ref.check(again, (f, d_f + (ref.half(kind) + 16 * ref.U) * f.abs()), "out again")
    alone, none = dp.packed_activation_backward(d_out, packed, act)
    assert none is None and torch.equal(alone, d_x)
    return out, packed, d_x


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("act", ACTS)
def test_pack_activations(dp, act, kind):
    g = gen(1)
    x = normal(g, 70, 520, dtype=TYPES[kind], std=2.0)
    check_pack(dp, x, act, normal(g, 70, 520, dtype=TYPES[kind]))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 7), (3, 8), (5, 127), (2, 128), (7, 129), (33, 1000), (300, 136), (1, 40000), (9, 4096), (40, 272)])
def test_pack_sizes(dp, rows, width, kind):
    g = gen(2)
    x = normal(g, rows, width, dtype=TYPES[kind])
    check_pack(dp, x, "gelu", normal(g, rows, width, dtype=TYPES[kind]))


@pytest.mark.parametrize("left,pad", [(0, 8), (1, 3), (8, 16)])
def test_pack_strides_and_leading_dimensions(dp, left, pad):
    g = gen(3)
    wide, wide_d = (normal(g, 6, 5, 256 + pad, dtype=torch.bfloat16) for _ in range(2))
    x, d_out = wide[..., min(left, pad):][..., :256], wide_d[..., min(left, pad):][..., :256]
    out, packed, d_x = check_pack(dp, x, "tanh", d_out)
    same = dp.activate_and_pack(x.contiguous(), "tanh")
    assert out.shape == (6, 5, 256) and packed.scales.shape == (6, 5, 2)
    assert torch.equal(out, same[0]) and torch.equal(packed.codes, same[1].codes)


@pytest.mark.parametrize("act", ACTS)
def test_pack_infinities_and_nan_show(dp, act):
    x = normal(gen(4), 6, 300)
    x[1, 5], x[2, 140], x[3, 299], x[4] = float("nan"), float("inf"), -float("inf"), 0.0
    x[5, :128] = 2.0 ** -101  # below what a block can hold
    out, packed = dp.activate_and_pack(x, act)
    codes, scales = ref.pack_reference(x)
    assert torch.equal(packed.codes.cpu(), codes)
    assert torch.equal(packed.scales.cpu().isnan(), scales.isnan())
    values = packed.unpack()
    d_x, again = dp.packed_activation_backward(torch.ones_like(x), packed, act, recompute=True)
    for row, block in ((1, 0), (2, 1), (3, 2)):
        for t in (values, d_x, again):
            part = t[row].split(128)
            assert part[block].isnan().all() and all(p.isfinite().all() for i, p in enumerate(part) if i != block)
    assert not values[4].any() and not values[5, :128].any()


def test_pack_no_rows(dp):
    x = torch.empty(0, 130, device="cuda")
    out, packed = dp.activate_and_pack(x, dp.GeLU())
    assert packed.codes.shape == (0, 130) and packed.scales.shape == (0, 2) and packed.unpack().shape == (0, 130)
    assert dp.packed_activation_backward(x, packed, dp.GeLU())[0].shape == (0, 130)


# ------------------------------------------------------------------------------ streams, graphs, repetition
def one_step(dp, t):
    """Forward and backward of a block and of the head; every output."""
    new, normed, stats = dp.residual_norm(t["x"], t["y"], gate=t["gate"], post_weight=t["wp"], pre_weight=t["wn"])
    out, packed = dp.activate_and_pack(normed, "gelu")
    loss, lse = dp.vocab_cross_entropy(out, t["head"], t["targets"])
    head = dp.vocab_cross_entropy_backward(t["grad"], out, t["head"], t["targets"], lse)
    d_normed, again = dp.packed_activation_backward(head.hidden, packed, "gelu", recompute=True)
    block = dp.residual_norm_backward(d_normed, None, new, t["y"], stats, gate=t["gate"], post_weight=t["wp"],
                                      pre_weight=t["wn"])
    return [new, normed, stats, out, packed.codes, packed.scales, loss, lse, head.hidden, head.weight, d_normed, again,
            *(g for g in block if g is not None)]


def step_inputs(seed, rows=200, width=264, vocab=1500, kind=torch.bfloat16):
    g = gen(seed)
    return dict(x=normal(g, rows, width, dtype=kind), y=normal(g, rows, width, dtype=kind),
                gate=normal(g, 4, width, dtype=kind, mean=1.0), wp=normal(g, width, dtype=kind, mean=1.0),
                wn=normal(g, width, dtype=kind, mean=1.0), head=normal(g, vocab, width, dtype=kind, std=0.1),
                targets=torch.randint(-1, vocab, (rows,), generator=g, device="cuda"),
                grad=torch.full((1,), 1.0 / rows, device="cuda"))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_same_inputs_same_bits(dp, kind):
    t = step_inputs(1, kind=TYPES[kind])
    first = one_step(dp, t)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, one_step(dp, t)))


def test_streams_at_once(dp):
    inputs = [step_inputs(s) for s in range(3)]
    want = [one_step(dp, t) for t in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [None] * 3
    for _ in range(4):
        for i, (s, t) in enumerate(zip(streams, inputs)):
            with torch.cuda.stream(s):
                got[i] = one_step(dp, t)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_and_replayed(dp):
    held, other = step_inputs(5), step_inputs(6)
    want = [one_step(dp, held), one_step(dp, other)]
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        outputs = one_step(dp, held)
    fresh = {k: v.clone() for k, v in held.items()}
    for new, expected in ((other, want[1]), (fresh, want[0])):
        for k, v in held.items():
            v.copy_(new[k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outputs, expected))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_training_step_of_a_residual_stack(dp, kind):
    """Three blocks (norm, linear, activation, linear, post norm, gate) and a head, forward and backward through the
    operators with torch's products between them, against automatic differentiation in 64 bits."""
    kind = TYPES[kind]
    g, rows, width, inner, vocab, blocks = gen(20), 96, 128, 256, 1003, 3
    p = dict(head=normal(g, vocab, width, dtype=kind, std=1.0 / width ** 0.5), final=normal(g, width, dtype=kind, std=0.1, mean=1.0))
    for i in range(blocks):
        p[f"up{i}"] = normal(g, inner, width, dtype=kind, std=1.0 / width ** 0.5)
        p[f"down{i}"] = normal(g, width, inner, dtype=kind, std=1.0 / inner ** 0.5)
        p[f"pre{i}"], p[f"post{i}"] = (normal(g, width, dtype=kind, std=0.1, mean=1.0) for _ in range(2))
        p[f"gate{i}"] = normal(g, width, dtype=kind, std=0.1, mean=0.5)
    x = normal(g, rows, width, dtype=kind)
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    targets[::7] = -100
    weight = torch.full((), 1.0 / int((targets >= 0).sum()), device="cuda")

    # forward
    stream, normed, stats = dp.residual_norm(x, norm="layer", pre_weight=p["pre0"])
    saved = []
    for i in range(blocks):
        pre = normed @ p[f"up{i}"].T
        out, packed = dp.activate_and_pack(pre, dp.GeLU())
        branch = out @ p[f"down{i}"].T
        after = p[f"pre{i + 1}"] if i + 1 < blocks else p["final"]
        step = dict(norm="layer", post_weight=p[f"post{i}"], gate=p[f"gate{i}"], branch_scale=0.5, pre_weight=after)
        before = normed
        stream, normed, stats = dp.residual_norm(stream, branch, **step)
        saved.append((before, packed, branch, stream, stats, step))
    loss, lse = dp.vocab_cross_entropy(normed, p["head"], targets)
    # backward
    grads = {}
    d_head = dp.vocab_cross_entropy_backward(weight, normed, p["head"], targets, lse)
    grads["head"], d_normed, d_stream = d_head.weight, d_head.hidden, None
    for i in reversed(range(blocks)):
        before, packed, branch, stream, stats, step = saved[i]
        b = dp.residual_norm_backward(d_normed, d_stream, stream, branch, stats, **step)
        grads[f"pre{i + 1}" if i + 1 < blocks else "final"] = b.pre_weight
        grads[f"post{i}"], grads[f"gate{i}"], d_stream = b.post_weight, b.gate, b.stream
        d_pre, out = dp.packed_activation_backward(b.branch @ p[f"down{i}"], packed, "gelu", recompute=True)
        grads[f"down{i}"], grads[f"up{i}"] = b.branch.T @ out, d_pre.T @ before
        d_normed = d_pre @ p[f"up{i}"]
    _, _, first_stats = dp.residual_norm(x, norm="layer", pre_weight=p["pre0"])
    b = dp.residual_norm_backward(d_normed, d_stream, x, None, first_stats, norm="layer", pre_weight=p["pre0"])
    grads["pre0"], grads["x"] = b.pre_weight, b.stream

    wide = {k: v.double().requires_grad_() for k, v in dict(p, x=x).items()}
    norm = lambda v: torch.nn.functional.layer_norm(v, (width,), eps=1e-6)  # noqa: E731
    r = wide["x"]
    for i in range(blocks):
        h = norm(r) * wide[f"pre{i}"]
        y = torch.nn.functional.gelu(h @ wide[f"up{i}"].T, approximate="tanh") @ wide[f"down{i}"].T
        r = r + 0.5 * wide[f"gate{i}"] * norm(y) * wide[f"post{i}"]
    logits = (norm(r) * wide["final"]) @ wide["head"].T
    keep = targets >= 0
    want = torch.nn.functional.cross_entropy(logits[keep], targets[keep], reduction="none")
    (want.sum() * weight.double()).backward()
    # Forward: a dozen stored values between input and loss, half a step each, that the norms neither
    # shrink nor grow: relative 12 * half in a vector of logits of deviation 1.  Gradients: besides as many
    # roundings, x is off by 1/254 of its block's largest (2.8 deviations of 128 normals) at most, uniformly:
    # 2.8 / 254 / sqrt(3) = 0.0064 deviations, which moves f and f' (slopes 1.1 and 0.8 at most) by that much;
    # three blocks add in squares, twice (f and f'): 0.0064 * sqrt(6) = 0.016; twice that is allowed.
    half = ref.half(kind)
    assert (loss[keep].double() - want).abs().max() < 4 * 12 * half + 1e-4
    assert not loss[~keep].any()
    for name, got in grads.items():
        value = wide[name].grad
        off = (got.double() - value).norm() / value.norm()
        assert off < 0.032 + 24 * half, (name, float(off))
