"""Calls of the operators (deepity_b200/operators.py) at the edge of what their documentation allows: infinities, host threads,
the largest sizes, waits that run out, and how exact 32-bit tensors are."""
import ctypes
import threading

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


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


# ------------------------------------------------------------------------------ infinities in operands
def infinite_case(rows, kind, seed=0):
    """The last word's weight holds -inf at column 3, where every row of hidden is positive: its logits are -inf."""
    g = gen(seed)
    hidden, weight = normal(g, rows, 40, dtype=kind), normal(g, 301, 40, dtype=kind, std=0.3)
    hidden[:, 3] = hidden[:, 3].abs() + 0.1
    weight[300, 3] = -float("inf")
    return hidden, weight, torch.randint(0, 300, (rows,), generator=g, device="cuda")


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [2, 5, 8, 9, 40, 300])
def test_infinite_weight_takes_its_word_out(dp, rows, kind):
    hidden, weight, targets = infinite_case(rows, TYPES[kind])
    grad = torch.linspace(0.5, 2.0, rows, device="cuda")
    want = ref.vocab_reference(hidden, weight[:300], targets, None, 1.0, -100, grad)
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets)
    ref.check(loss, want["loss"], "loss")
    ref.check(lse, want["lse"], "lse")
    got = dp.vocab_cross_entropy_backward(grad, hidden, weight, targets, lse)
    ref.check(got.weight[:300], want["weight"], "d_weight")
    assert not got.weight[300].any()
    keep = torch.arange(40, device="cuda") != 3
    value, bound = want["hidden"]
    ref.check(got.hidden[:, keep], (value[:, keep], bound[:, keep]), "d_hidden")
    assert got.hidden[:, 3].isnan().all()  # 0 * inf


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [2, 5, 40])
def test_infinite_logits_follow_the_signs(dp, rows, kind):
    hidden, weight, targets = infinite_case(rows, TYPES[kind], seed=1)
    clean = dp.vocab_cross_entropy(hidden, weight, targets)
    moved = hidden.clone()
    moved[0, 3], moved[1, 3] = -0.5, 0.0  # +inf among the logits; 0 * inf
    loss, lse = dp.vocab_cross_entropy(moved, weight, targets)
    assert not loss[:2].isfinite().any() and not lse[:2].isfinite().any()
    assert torch.equal(loss[2:], clean[0][2:]) and torch.equal(lse[2:], clean[1][2:])
    targets[0] = 300  # the word that is out: its loss is infinite, the others stay
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets)
    assert loss[0] == float("inf") and torch.equal(lse, clean[1]) and torch.equal(loss[1:], clean[0][1:])
    got = dp.vocab_cross_entropy_backward(torch.ones(1, device="cuda"), hidden, weight, targets, lse)
    assert got.hidden[0, 3].isnan() or got.hidden[0, 3] == float("inf")
    assert got.weight.isfinite().all()


def test_infinite_hidden_stays_in_its_row(dp):
    hidden, weight, targets = infinite_case(70, torch.float32, seed=2)
    weight[300, 3] = 0.25
    clean = dp.vocab_cross_entropy(hidden, weight, targets)
    hidden[7, 3] = float("inf")  # times weights of both signs
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets)
    assert not loss[7].isfinite() and not lse[7].isfinite()
    keep = torch.arange(70, device="cuda") != 7
    assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(lse[keep], clean[1][keep])
    weight[:, 3] = -weight[:, 3].abs() - 0.01  # all logits are -inf
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets)
    assert lse[7] == -float("inf") and loss[7].isnan()


@pytest.mark.parametrize("rows", [5, 40])
def test_numbers_above_the_largest_bf16(dp, rows):
    """The largest float32 numbers round to an infinity in bf16 and are none themselves."""
    g = gen(3)
    hidden, weight = normal(g, rows, 40), normal(g, 300, 40, std=0.3)
    hidden, weight = hidden * 2.0 ** -10, weight * 2.0 ** 40
    hidden[:, 3] = 2.0 ** -100
    weight[:, 3] = torch.linspace(-1.0, 1.0, 300, device="cuda") * torch.finfo(torch.float32).max
    targets = torch.randint(0, 300, (rows,), generator=g, device="cuda")
    scale = 2.0 ** -27  # logits up to 2^128 * 2^-100 * 2^-27 = 2
    want = ref.vocab_reference(hidden, weight, targets, None, scale, -100)
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, scale=scale)
    ref.check(loss, want["loss"], "loss")
    ref.check(lse, want["lse"], "lse")


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_ignored_rows_have_no_gradient_whatever_the_weights_hold(dp, kind):
    hidden, weight, targets = infinite_case(150, TYPES[kind], seed=4)
    targets[3], targets[77], targets[149] = -100, 301, -1
    for bad in (float("inf"), float("nan")):
        weight[20, 5] = bad
        loss, lse = dp.vocab_cross_entropy(hidden, weight, targets)
        got = dp.vocab_cross_entropy_backward(torch.ones(1, device="cuda"), hidden, weight, targets, lse)
        for row in (3, 77, 149):
            assert loss[row] == 0 and lse[row] == 0 and not got.hidden[row].any()


@pytest.mark.parametrize("kind,rows,width,vocab", [("f32", 9, 2048, 30000), ("f32", 300, 2048, 50000), ("bf16", 300, 1021, 140001)])
def test_vocab_forward_in_pieces(dp, kind, rows, width, vocab):
    """Weights whose copies take more than 256 MB come in pieces: bias, targets and partial sums of the later ones too.  (9 rows: one more
    than the kernel for few rows takes.)"""
    kind, g = TYPES[kind], gen(rows)
    hidden, weight = normal(g, rows, width, dtype=kind), normal(g, vocab, width, dtype=kind, std=2.0 / width ** 0.5)
    bias = normal(g, vocab, dtype=kind)
    assert vocab * width * (6 if kind == torch.float32 else 2) > 256 << 20
    targets = torch.randint(vocab // 2, vocab, (rows,), generator=g, device="cuda")
    targets[0], targets[1], targets[2] = vocab - 1, 0, -100
    want = ref.vocab_reference(hidden, weight, targets, bias, 0.5, -100)
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias, scale=0.5)
    ref.check(loss, want["loss"], "loss")
    ref.check(lse, want["lse"], "lse")
    # the bounds above are wide; exponentials (2^-22) and logits of |l| <= 10 to 2^-18 (64 truncating additions) leave 4e-5 at most
    assert (loss.double() - want["loss"][0]).abs().max() < 4e-5 and (lse.double() - want["lse"][0]).abs().max() < 4e-5


def test_vocab_sums_are_shared_out_by_the_tiles_there_are(dp):
    """d_hidden's contraction is shared out so that rounds * (1 + 3 % a share) is least, with the tiles that are launched: 128 columns
    each for float32.  How many shares there are shows in the workspace, where each has its sums."""
    from deepity_b200 import _lib
    lib, size = _lib.load(), ctypes.c_size_t()
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    up = lambda v, to: -(-v // to) * to  # noqa: E731
    for rows, width, vocab in ((777, 515, 10007), (777, 641, 10007), (2048, 1100, 8000), (300, 130, 2000)):
        c = _lib.VocabCe(rows=rows, width=width, vocab=vocab, hidden_stride=width, weight_stride=width, type=0, scale=1.0,
                         d_hidden_stride=width, d_weight_stride=width)
        _lib.check(lib.dpc_vocab_ce_workspace(ctypes.byref(c), 1, ctypes.byref(size)))
        copies = 6 * up(width, 8)  # three planes of a row
        rest = 256 + up(rows * copies, 256) + up(vocab * copies, 256) + up(rows * up(vocab, 256) * 6, 256)
        sums = rows * up(width, 256) * 4
        shares = (size.value - rest) // sums
        tiles, blocks = -(-rows // 256) * -(-width // 128), -(-vocab // 64)
        cost = {n: -(-tiles * n // pairs) / n * (1 + 0.03 * n) for n in range(1, max(1, min(pairs, blocks // 4)) + 1)}
        assert size.value == rest + up(shares * sums, 256) and cost[shares] == min(cost.values()), (rows, width, shares)


# ------------------------------------------------------------------------------ packed activations
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_tanh_is_exact_relative_to_its_value(dp, kind):
    """Small and large arguments, and both sides of every border between the forms; the kept values' too.

    Errors relative to tanh: a polynomial with 3 roundings, or (1 - e) / (1 + e) with e = exp(-2 |x|) <= 0.37: e is off by 2^-22 of itself
    and by the rounding of its exponent, 2 |x| log2(e) U < 0.1 * 2^-22 in all, which moves tanh by 1.2 * 0.37 * 2^-22 / 0.46 of
    itself, a reciprocal is off by 2^-23 and 4 roundings by U each: below 2^-20 together.  The slope 4 e / (1 + e)^2 takes over e's own
    relative error, 2^-22 + 3 |x| U, two reciprocals and 4 roundings: below 2^-20 + |x| 2^-22; 1 - tanh^2 >= 0.75 loses nothing.
    For bf16 tensors the border is 1/16: the third term of the series is left out, 2 x^4 / 15 < 2^-18, and above it e's error of
    2^-22 moves tanh by 0.5 * 2^-22 / 0.062 = 2^-18 of itself: 2^-17."""
    kind, g = TYPES[kind], gen(5)
    e = 2.0 ** -20 if kind == torch.float32 else 2.0 ** -17
    size = 10.0 ** torch.linspace(-30, 1.6, 128 * 128, device="cuda").view(128, 128)
    border = torch.cat([torch.linspace(at - 0.001, at + 0.001, 128, device="cuda").expand(4, 128) for at in (0.5, 0.0625)])
    x = torch.cat([size, border, normal(g, 60, 128)])
    x = torch.cat([x, -x]).to(kind)
    out, packed = dp.activate_and_pack(x, "tanh")
    want = x.double().tanh()
    ref.check(out, (want, (e + ref.half(kind)) * want.abs()), "out")
    d_x, again = dp.packed_activation_backward(torch.ones_like(x), packed, "tanh", recompute=True)
    kept = packed.unpack().double()
    want = kept.tanh()
    ref.check(again, (want, (e + ref.half(kind)) * want.abs()), "out again")
    slope = 1.0 / kept.cosh().square()
    ref.check(d_x, (slope, (e + kept.abs() * 2.0 ** -22 + ref.half(kind)) * slope + 2.0 ** -126), "d_preact")
    x[0, 0], x[1, 0], x[2, 0] = float("nan"), float("inf"), -float("inf")
    out = dp.activate_and_pack(x, "tanh")[0]
    assert out[0, 0].isnan() and out[1, 0] == 1 and out[2, 0] == -1


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_esigmoid_is_exact_relative_to_its_value(dp, kind):
    """0.5 / (1 + |x|) on the left of 0 and 1 less that on the right: the sum, a reciprocal good to 2^-23 and a difference or a square, below
    2^-21 of the value together."""
    kind = TYPES[kind]
    x = 10.0 ** torch.linspace(-6, 30, 64 * 128, device="cuda").view(64, 128)
    x = torch.cat([x, -x]).to(kind)
    out, packed = dp.activate_and_pack(x, "esigmoid")
    half = lambda v: 0.5 / (1 + v.double().abs())  # noqa: E731
    want = torch.where(x < 0, half(x), 1 - half(x))
    ref.check(out, (want, (2.0 ** -21 + ref.half(kind)) * want), "out")
    d_x, again = dp.packed_activation_backward(torch.ones_like(x), packed, "esigmoid", recompute=True)
    kept = packed.unpack()
    want = torch.where(kept < 0, half(kept), 1 - half(kept))
    ref.check(again, (want, (2.0 ** -21 + ref.half(kind)) * want), "out again")
    slope = 2 * half(kept) ** 2
    ref.check(d_x, (slope, (2.0 ** -21 + ref.half(kind)) * slope + 2.0 ** -126), "d_preact")
    x[0, 0], x[1, 0], x[2, 0] = float("nan"), float("inf"), -float("inf")
    out = dp.activate_and_pack(x, "esigmoid")[0]
    assert out[0, 0].isnan() and out[1, 0] == 1 and out[2, 0] == 0


# ------------------------------------------------------------------------------ host threads
def at_once(*works):
    """Every work on a thread and a stream of its own; what they raised."""
    raised = []

    def call(work):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                work()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 (handed to the test)
            raised.append(e)

    threads = [threading.Thread(target=call, args=(w,)) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return raised


def test_host_threads_with_norms_of_two_widths(dp):
    """One kernel, whose shared memory goes by the width: neither thread may take it from the other."""
    def steps(width):
        def work():
            g = gen(width)
            x, w = normal(g, 64, width, dtype=torch.bfloat16), normal(g, width, dtype=torch.bfloat16)
            _, h, stats = dp.residual_norm(x, pre_weight=w)
            want = dp.residual_norm_backward(h, None, x, None, stats, pre_weight=w)
            for _ in range(3000):
                got = dp.residual_norm_backward(h, None, x, None, stats, pre_weight=w)
            assert torch.equal(got.stream, want.stream) and torch.equal(got.pre_weight, want.pre_weight)
        return work

    assert at_once(*(steps(width) for width in (4104, 8192, 4104, 8192))) == []


def test_host_threads_with_few_rows_of_two_widths(dp):
    def steps(width):
        def work():
            g = gen(width)
            hidden, weight = normal(g, 5, width), normal(g, 50, width)
            targets = torch.arange(5, device="cuda")
            want = dp.vocab_cross_entropy(hidden, weight, targets)[0]
            for _ in range(3000):
                got = dp.vocab_cross_entropy(hidden, weight, targets)[0]
            assert torch.equal(got, want)
        return work

    assert at_once(*(steps(width) for width in (256, 2304, 256, 2304))) == []


# ------------------------------------------------------------------------------ the smallest and the largest sizes
def test_norm_of_no_sequences_with_a_gate_each(dp):
    empty, gate, weight = torch.empty(0, 7, 40, device="cuda"), torch.empty(0, 40, device="cuda"), torch.ones(40, device="cuda")
    new, normed, stats = dp.residual_norm(empty, empty, gate=gate, pre_weight=weight)
    got = dp.residual_norm_backward(empty, None, new, empty, stats, gate=gate, pre_weight=weight)
    assert new.shape == normed.shape == got.stream.shape == (0, 7, 40) and got.gate.shape == (0, 40)
    assert got.pre_weight.shape == (40,) and not got.pre_weight.any()
    with pytest.raises(ValueError, match="gate"):
        dp.residual_norm(torch.ones(2, 40, device="cuda"), torch.ones(2, 40, device="cuda"), gate=gate)


def test_norm_gradient_of_the_most_rows(dp):
    """2^31 - 1 rows, each a group of its own: the last ones' gradients are those of a call with them alone, and the others' are 0."""
    torch.cuda.empty_cache()
    rows, few, g = (1 << 31) - 1, 9, gen(6)
    big = {k: torch.zeros(rows, 1, device="cuda", dtype=torch.bfloat16) for k in ("new", "branch", "gate", "d_normed")}
    for t in big.values():
        t[-few:] = normal(g, few, 1, dtype=torch.bfloat16)
    stats = torch.zeros(rows, 4, device="cuda")
    stats[-few:] = normal(g, few, 4)
    last = {k: t[-few:].clone() for k, t in big.items()}

    def gradients(t, stats):
        got = dp.residual_norm_backward(t["d_normed"], None, t["new"], t["branch"], stats, gate=t["gate"])
        return got.stream, got.branch, got.gate

    want = gradients(last, stats[-few:].clone())
    for a, b in zip(gradients(big, stats), want):
        assert torch.equal(a[-few:], b) and not a[:-few].any()
    del big, stats, a
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------ waits that run out
def entry(name, c, backward=None):
    """A C entry on torch's current stream, with a workspace of its own."""
    from deepity_b200 import _lib
    lib, size, more = _lib.load(), ctypes.c_size_t(), () if backward is None else (backward,)
    _lib.check(getattr(lib, name + "_workspace")(ctypes.byref(c), *more, ctypes.byref(size)))
    held = torch.empty(size.value, device="cuda", dtype=torch.uint8)
    c.workspace, c.workspace_bytes = held.data_ptr(), size.value
    call = name + ("_forward" if backward == 0 else "_backward")
    _lib.check(getattr(lib, call)(torch.cuda.current_stream().cuda_stream, ctypes.byref(c)))
    torch.cuda.synchronize()


@pytest.fixture
def wait_limit(built_library):
    """wait_limit(1): 2 ms, and a signal is kept back; wait_limit(0): as it was, and so at the test's end."""
    from deepity_b200 import _lib

    def to(keep_back):
        _lib.check(_lib.load().dpc_operators_set_wait_limit(2.0 * keep_back, keep_back))

    yield to
    to(0)


@pytest.mark.parametrize("kind,rows,width,vocab", [("bf16", 40, 64, 300), ("bf16", 700, 264, 40001), ("f32", 40, 64, 300),
                                                   ("f32", 300, 1100, 5003)])
def test_vocab_waits_that_run_out_leave_nan(dp, wait_limit, kind, rows, width, vocab):
    """A signal is kept back: after 2 ms the kernels give up and return, and what was not computed is NaN.  The next call is right."""
    from deepity_b200 import _lib
    g, kind = gen(7), TYPES[kind]
    hidden, weight, bias = normal(g, rows, width, dtype=kind), normal(g, vocab, width, dtype=kind), normal(g, vocab, dtype=kind)
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    targets[5], targets[-1] = -100, vocab
    counted = (targets >= 0) & (targets < vocab)
    one = torch.ones(1, device="cuda")
    loss, lse = dp.vocab_cross_entropy(hidden, weight, targets, bias)
    want = dp.vocab_cross_entropy_backward(one, hidden, weight, targets, lse, bias)
    for keep_back in (1, 0):
        out = {k: torch.full_like(t, 7.0) for k, t in dict(loss=loss, lse=lse, hidden=hidden, weight=weight, bias=bias).items()}
        c = _lib.VocabCe(rows=rows, width=width, vocab=vocab, hidden_stride=width, weight_stride=width,
                         type=0 if kind == torch.float32 else 1, scale=1.0, ignore_index=-100, hidden=hidden.data_ptr(),
                         weight=weight.data_ptr(), bias=bias.data_ptr(), targets=targets.data_ptr(), loss=out["loss"].data_ptr(),
                         lse=out["lse"].data_ptr())
        wait_limit(keep_back)
        entry("dpc_vocab_ce", c, 0)
        c.lse, c.grad_loss, c.grad_stride = lse.data_ptr(), one.data_ptr(), 0
        c.d_hidden, c.d_hidden_stride, c.d_weight, c.d_weight_stride = out["hidden"].data_ptr(), width, out["weight"].data_ptr(), width
        c.d_bias = out["bias"].data_ptr()
        entry("dpc_vocab_ce", c, 1)
        if keep_back:
            for name in ("loss", "lse", "hidden"):
                assert out[name][counted].isnan().all() and not out[name][~counted].any(), name
            assert out["weight"].isnan().all() and out["bias"].isnan().all()
        else:
            assert torch.equal(out["loss"], loss) and torch.equal(out["lse"], lse)
            assert all(torch.equal(out[name], getattr(want, name)) for name in ("hidden", "weight", "bias"))


@pytest.mark.parametrize("kind,rows,width,waits", [("bf16", 3, 256, True), ("bf16", 900, 256, True), ("bf16", 900, 4096, True),
                                                   ("f32", 900, 2048, True), ("bf16", 9, 12288, True), ("bf16", 9, 16384, False),
                                                   ("bf16", 9, 255, False)])
def test_norm_waits_that_run_out_leave_nan(dp, wait_limit, kind, rows, width, waits):
    """(Two rows ahead of 16384 in bf16 take 4 * 2 * 2 * 16384 bytes, more than an SM's shared memory, and rows off 16 bytes are not
    fetched ahead: no waits.)"""
    from deepity_b200 import _lib
    g, kind = gen(8), TYPES[kind]
    x, y, d = (normal(g, rows, width, dtype=kind) for _ in range(3))
    vectors = {k: normal(g, width, dtype=kind) for k in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias")}
    new, _, stats = dp.residual_norm(x, y, norm="layer", **vectors)
    want = dp.residual_norm_backward(d, None, new, y, stats, norm="layer", **vectors)
    for keep_back in (1, 0):
        out = {k: torch.full_like(t, 7.0) for k, t in dict(vectors, stream=x, branch=y).items()}
        c = _lib.ResidualNorm(rows=rows, width=width, groups=1, type=0 if kind == torch.float32 else 1, norm=1, post_norm=1,
                              stream_scale=1.0, branch_scale=1.0, branch=y.data_ptr(), branch_stride=width, gate_stride=width,
                              new_stream=new.data_ptr(), new_stream_stride=width, stats=stats.data_ptr(), d_normed=d.data_ptr(),
                              d_normed_stride=width, d_stream_stride=width, d_branch_stride=width, d_gate_stride=width,
                              **{k: v.data_ptr() for k, v in vectors.items()}, **{"d_" + k: v.data_ptr() for k, v in out.items()})
        wait_limit(keep_back)
        entry("dpc_residual_norm", c)
        for name, t in out.items():
            assert t.isnan().all() if keep_back and waits else torch.equal(t, getattr(want, name)), name
