"""The operators' calls at the ends of what their documentation allows, against their definitions in 64 bits: norms without an eps, weights and positions at the ends of their
types' ranges, long sums, outputs that share memory with inputs."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
U = {t: torch.finfo(t).eps / 2 for t in TYPES}
E = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    from radzero_amd import ops
    return ops


def randn(seed, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * std).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("shape", [(1, 300), (8, 300), (20, 300), (200, 300), (1, 9000), (3, 9000), (20, 9000), (200, 9000)], ids=str)
def test_diff_attention_of_hidden_rows_without_an_eps(ops, dtype, d, shape):
    """norm_eps = 0: a query that sees no key still gets zeros (an empty sequence, a mask of nothing, causal rows before the first key), whole and in pieces; the others what
    an eps far below their mean square gives, and NaN stays NaN."""
    n_q, n_k = shape
    b, h = 4, 2
    q, k, v = randn(1, b, n_q, h, 2 * d, dtype=dtype), randn(2, b, n_k, h, 2 * d, dtype=dtype), randn(3, b, n_k, h, 2 * d, dtype=dtype) + 1
    lam, w = torch.zeros(4, d, device="cuda"), torch.ones(2 * d, device="cuda")
    mask = torch.ones(b, n_k, dtype=torch.int64, device="cuda")
    mask[1] = 0
    lens = torch.tensor([0, n_k, n_q // 2, n_k], dtype=torch.int32, device="cuda")
    for kv_lens in (None, lens):
        for causal in (None, "end"):
            call = lambda eps: ops.diff_attention(q, k, v, lam, lambda_init=0.3, causal=causal, kv_lens=kv_lens, attention_mask=mask, norm_weight=w, norm_eps=eps)      # noqa: E731
            got = call(0.0)
            n = torch.full((b,), n_k, device="cuda") if kv_lens is None else kv_lens.long()
            n[1] = 0
            sees = (n[:, None] > 0) & ((n[:, None] - n_q + torch.arange(n_q, device="cuda") >= 0) if causal else torch.ones(1, n_q, dtype=torch.bool, device="cuda"))
            assert bool((got[~sees] == 0).all()), (kv_lens is not None, causal)
            assert bool(torch.isfinite(got.float()).all())
            # a mean square is at least 1e-6 here (values of mean 1, 1 - lambda = 0.7): 1e-30 beside it changes nothing
            assert torch.equal(got, call(1e-30))
    k[3, 0, 0, 0] = math.nan
    got = ops.diff_attention(q, k, v, lam, lambda_init=0.3, attention_mask=mask, norm_weight=w, norm_eps=0.0)
    assert bool(got[3, :, 0].isnan().all()) and bool((got[1] == 0).all()) and bool(torch.isfinite(got[3, :, 1].float()).all())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("at", [0, 30000, 65535])
@pytest.mark.parametrize("below", [20.03, 25.05, 28.0])
@pytest.mark.parametrize("shape", [(512, 3), (600, 64)], ids=str)
def test_diff_attention_one_key_above_a_flat_tail(ops, dtype, at, below, shape):
    """One key, and 65535 whose weights are 2^-below of its own each: their share of the sum is kept, whether a query's keys are in one piece or several.

    Bounds.  A weight is rounded by at most u of it, or, in f16, whose steps end at 2^-24, by 2^-25 on a scale that puts the largest weight at 2^4 or above for 65536 keys:
    2^16 2^-29 = 2^-13 of the sum.  That and the sum's own rounding (n / 16 additions of fp32 at worst) count in the values' sum and in the weights' sum: twice.  The scores'
    exponents are below 32 and off by 2 E of them."""
    units, n_q = shape
    d, n = 64, 1 << 16
    q, k, v = (torch.zeros(x, 1, 2 * d, device="cuda", dtype=dtype) for x in (n_q, n, n))
    q[:, 0, 0] = 8
    k[at, 0, 0] = below * math.log(2)
    v[:] = 1
    v[at, 0, :32], v[:, 0, 32:64] = 0, 0
    v[at, 0, 32:64] = 1
    got = ops.diff_attention(*(x.expand(units, -1, -1, -1) for x in (q, k, v)), torch.zeros(4, d, device="cuda"), lambda_init=0.0, scale=1 / 8).double()
    tail = (n - 1) * math.exp(-float(k[at, 0, 0].double()))
    head, tail = 1 / (1 + tail), tail / (1 + tail)
    u = U[dtype] if dtype != torch.float32 else 0.0
    for columns, ref in ((slice(0, 32), tail), (slice(32, 64), head), (slice(64, 128), 1.0)):
        off = 2 * (u * tail + (2.0 ** -13 if dtype == torch.float16 else 0)) if ref != 1.0 else 0
        tol = off + 2 * n / 16 * E * ref + 128 * E * tail + U[dtype] * ref + 2.0 ** -25
        assert float((got[..., columns] - ref).abs().max()) <= tol, (columns, ref, got[..., columns].min(), got[..., columns].max(), tol)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 4, 8, 12, 32, 70])
def test_diff_attention_fp32_of_equal_values(ops, d, rows):
    """65536 equal scores (every weight is 1) and equal values of 1 + 2^-12, keys not split over workgroups: the mean is the value.

    Whatever the sums' size, a form may round them once for 32 keys, by half a step at most: n / 32 times E of the result, if every rounding went the same way.  Adding fewer keys
    at a time does that here: the value's last bit falls off the sum each time."""
    n, units, value = 1 << 16, 1100, 1 + 2.0 ** -12
    q, k, v = torch.zeros(1, rows, 1, 2 * d, device="cuda"), torch.zeros(1, n, 1, 2 * d, device="cuda"), torch.full((1, n, 1, 2 * d), value, device="cuda")
    got = ops.diff_attention(*(x.expand(units, -1, -1, -1) for x in (q, k, v)), torch.zeros(4, d, device="cuda"), lambda_init=0.0)
    assert float((got.double() / value - 1).abs().max()) <= n / 32 * E


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 4, 8, 12, 32, 70])
def test_diff_attention_fp32_over_many_keys_of_few_rows(ops, d, rows):
    """The root mean square error of fp32 over 6000 keys, most sequences' by one workgroup alone.  One rounding of at most half a step at the sum's size for 32 keys, going either way:
    sqrt(n / 32) of them in a sum, in the values' and in the weights' one: sqrt(2); lambda is 0, so that nothing cancels."""
    n, units = 6000, 1100
    q, k = randn(1, 1, rows, 1, 2 * d), randn(2, 1, n, 1, 2 * d)
    v = randn(3, 1, n, 1, 2 * d) + 1
    got = ops.diff_attention(*(x.expand(units, -1, -1, -1) for x in (q, k, v)), torch.zeros(4, d, device="cuda"), lambda_init=0.0)
    p = torch.softmax(q[0, :, 0, :d].double() @ k[0, :, 0, :d].double().t().contiguous() / math.sqrt(d), -1)
    ref = p @ v[0, :, 0].double()
    # every sequence, whole or (the last ones) in pieces
    assert float((got[:, :, 0].double() - ref).flatten(1).norm(dim=1).max() / ref.norm()) <= math.sqrt(2) * math.sqrt(n / 32) * E


def block_calls(ops):
    """{operator: (call with a dict of changed arguments, its arguments)}, small."""
    h = randn(11, 2, 4, 64)
    args = {
        "rotary": dict(q=randn(1, 2, 4, 2, 64), k=randn(2, 2, 4, 2, 64), positions=torch.arange(4, device="cuda"), freqs=ops.rotary_frequencies(64, device="cuda")[0]),
        "diff_attention": dict(q=randn(3, 2, 4, 2, 64), k=randn(4, 2, 5, 2, 64), v=randn(5, 2, 5, 2, 64), lambda_qk=randn(6, 4, 32), lambda_init=0.3, norm_weight=randn(7, 64)),
        "residual_norm": dict(residual=h, y=randn(8, 2, 4, 64), pre_norm=ops.Norm(randn(9, 64), randn(10, 64)), post_norm=ops.Norm(randn(12, 64), randn(13, 64)), scale=randn(14, 64),
                              gate=randn(15, 2, 64)),
    }
    return {name: (lambda name=name, **change: getattr(ops, name)(**{**args[name], **change}), args[name]) for name in args}


INPUTS = [("rotary", n) for n in ("q", "k", "freqs")] + [("diff_attention", n) for n in ("q", "k", "v", "lambda_qk", "norm_weight")] + [
    ("residual_norm", n) for n in ("residual", "y", "scale", "gate", "pre_norm.weight", "pre_norm.bias", "post_norm.weight", "post_norm.bias")]


def changed(args, name, f):
    """{argument: itself with f applied to the tensor `name`}."""
    name, _, part = name.partition(".")
    return {name: args[name]._replace(**{part: f(getattr(args[name], part))}) if part else f(args[name])}


@pytest.mark.parametrize("operator,name", INPUTS, ids=lambda x: x)
def test_operators_refuse_every_input_that_asks_for_a_gradient(ops, operator, name):
    call, args = block_calls(ops)[operator]
    want = call()
    asking = changed(args, name, lambda t: t.clone().requires_grad_())
    with pytest.raises(ValueError, match="gradient"):
        call(**asking)
    with torch.no_grad():
        got = call(**asking)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("operator,name", INPUTS, ids=lambda x: x)
def test_operators_refuse_every_input_with_a_forward_derivative(ops, operator, name):
    call, args = block_calls(ops)[operator]
    want = call()
    with torch.autograd.forward_ad.dual_level():
        for x, y in zip(call(), want):                   # plain inputs inside such a level
            assert torch.equal(x, y)
        dual = changed(args, name, lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(ValueError, match="forward-mode"):
            call(**dual)


OUTPUTS = [("rotary", lambda a: ("q", "k")), ("diff_attention", lambda a: ("q",)), ("residual_norm", lambda a: ("residual", "y"))]


@pytest.mark.parametrize("operator,like", OUTPUTS, ids=lambda x: x if isinstance(x, str) else "")
def test_outputs_count_as_written_in_place(ops, operator, like):
    """A backward pass that saved a tensor before an operator wrote it raises, as it does for any in-place operation, also without grad mode; an output that asks for a gradient or
    carries a forward-mode one is refused."""
    call, args = block_calls(ops)[operator]
    given = lambda outs: outs[0] if operator == "diff_attention" else tuple(outs)      # noqa: E731
    names = like(args)
    for i in range(len(names)):
        outs = [torch.zeros_like(args[n]) for n in names]
        w = torch.ones((), device="cuda", requires_grad=True)
        loss = (outs[i] * w).sum()
        with torch.no_grad():
            got = call(out=given(outs))
        assert all(x is y for x, y in zip(outs, got if isinstance(got, tuple) else (got,)))
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
        outs[i] = outs[i].detach().requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            call(out=given(outs))
        with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
            outs[i] = torch.autograd.forward_ad.make_dual(torch.zeros_like(args[names[i]]), torch.ones_like(args[names[i]]))
            call(out=given(outs))
    with torch.inference_mode():
        outs = [torch.zeros_like(args[n]) for n in names]
        call(out=given(outs))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_residual_norm_over_its_residual_keeps_the_residual(ops, dtype):
    """x written where the residual stands, with nothing added to it: r still is the residual."""
    h = randn(21, 3, 5, 100, dtype=dtype)
    was, want = h.clone(), ops.residual_norm(h, pre_norm=ops.Norm())[1]
    r, x = ops.residual_norm(h, pre_norm=ops.Norm(), out=(None, h))
    assert x is h and torch.equal(x, want) and torch.equal(r, was)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_operators_refuse_outputs_that_overlap(ops, dtype):
    """Shifted, crossed, shared and differently laid out outputs; what lies between an input's rows, or is the input, is fine."""
    freqs = ops.rotary_frequencies(64, device="cuda")[0]
    packed = randn(31, 2, 9, 6, 64, dtype=dtype)
    q, k, v = packed[:, :, :2], packed[:, :, 2:4], packed[:, :, 4:]
    pos, lam = torch.arange(9, device="cuda"), torch.zeros(4, 32, device="cuda")
    turn = lambda *out: ops.rotary(q, k, positions=pos, freqs=freqs, out=out)      # noqa: E731
    h, y = (randn(s, 2, 8, 65, dtype=dtype) for s in (32, 33))
    norm = lambda *out: ops.residual_norm(h[:, 1:, :64], y[:, 1:, :64], pre_norm=ops.Norm(), out=out)      # noqa: E731
    before = packed.clone(), h.clone(), y.clone()
    for call in [lambda: turn(k, q), lambda: turn(v, v), lambda: turn(q, packed[:, :, 1:3]), lambda: turn(packed[:, :, 1:3], None), lambda: turn(None, q),
                 lambda: ops.diff_attention(q, k, v, lam, lambda_init=0.3, out=packed[:, :, 1:3]), lambda: ops.diff_attention(q, k, v, lam, lambda_init=0.3, out=v),
                 lambda: norm(h[:, :7, :64], None), lambda: norm(h[:, 1:, 1:], None), lambda: norm(None, y[:, 1:, 1:]), lambda: norm(h[:, 1:, :64], h[:, 1:, :64]),
                 lambda: norm(None, y[:, :7, :64])]:
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert torch.equal(packed, before[0]) and torch.equal(h, before[1]) and torch.equal(y, before[2])
    want = ops.diff_attention(q, k, k, lam, lambda_init=0.3)
    assert torch.equal(ops.diff_attention(q, k, k, lam, lambda_init=0.3, out=v), want)          # between the rows of q and k
    want = turn(None, None)
    got = turn(q, k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    want = norm(None, None)
    r, x = norm(y[:, 1:, :64], h[:, 1:, :64])            # each over the other input
    assert torch.equal(r, want[0]) and torch.equal(x, want[1])


def test_operators_refuse_arguments_beyond_their_fields(ops):
    """Sizes of 2^31 (views without memory of their own) and what is no number are refused like any other bad argument.  (A factor beyond float32 is an infinity, as it is there.)"""
    q, lam = torch.zeros(1, 1, 1, 64, device="cuda"), torch.zeros(4, 32, device="cuda")
    pos, freqs = torch.zeros(1, dtype=torch.int64, device="cuda"), ops.rotary_frequencies(64, device="cuda")[0]
    long, h = q.expand(1, 1 << 31, 1, 64), torch.zeros(2, 64, device="cuda")
    for call in [lambda: ops.diff_attention(q, long, long, lam, lambda_init=0.3), lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.3, out_scale=None),
                 lambda: ops.rotary(q, positions=pos, freqs=freqs, amplitude="2"), lambda: ops.residual_norm(h, h, pre_norm=None, alpha=10 ** 400)]:
        with pytest.raises(ValueError, match="Args"):
            call()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("axes", [1, 2])
def test_rotary_at_the_farthest_positions(ops, dtype, layout, axes):
    """One turn at positions from 2^24 to 2^31 of either sign, against cosines and sines of the angles in 64 bits.

    The angle's product is the same in both.  The kernel then takes turns = angle / (2 pi), off by 2 roundings (the factor's and the product's) of at most 2^-53 of 2^31 / (2 pi)
    turns: 2 2^-22 radian; the reference's cosine takes the angle as it is.  A fraction of a turn in fp32, its sine and cosine and three roundings: 5e-7."""
    x = randn(41, 2, 300, 3, 64, dtype=dtype)
    far = torch.randint(1 << 24, (1 << 31) - 1, (2, 300, axes), generator=torch.Generator(device="cuda").manual_seed(42), device="cuda")
    far[0, :6, 0] = torch.tensor([(1 << 31) - 1, 1 << 30, (1 << 30) + 1, (1 << 24) + 1, 16777219, 2147483629], device="cuda")
    far[1] *= -1
    freqs, _ = ops.rotary_frequencies(64, axes=axes, device="cuda")
    got = ops.rotary(x, positions=far if axes > 1 else far[..., 0], freqs=freqs, layout=layout).double()
    angle = (far.double()[..., None] * freqs.view(axes, -1)).flatten(-2)[:, :, None]
    pairs = (lambda t: (t[..., :32], t[..., 32:])) if layout == "half" else (lambda t: (t[..., 0::2], t[..., 1::2]))
    u, w = pairs(x.double())
    for y, ref in zip(pairs(got), (u * angle.cos() - w * angle.sin(), u * angle.sin() + w * angle.cos())):
        tol = (5e-7 + 2 * 2.0 ** -22) * (u.abs() + w.abs())
        tol = tol + U[dtype] * (ref.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert bool(((y - ref).abs() <= tol).all())


def test_operators_refuse_outputs_whose_rows_overlap(ops):
    q, lam = randn(51, 2, 9, 2, 64), torch.zeros(4, 32, device="cuda")
    pos, freqs = torch.arange(9, device="cuda"), ops.rotary_frequencies(64, device="cuda")[0]
    windows = torch.zeros(10000, device="cuda").as_strided(q.shape, (1152, 64, 64, 1))
    h = randn(52, 9, 64)
    for call in [lambda: ops.rotary(q, positions=pos, freqs=freqs, out=windows), lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.3, out=windows),
                 lambda: ops.residual_norm(h, pre_norm=ops.Norm(), out=(None, torch.zeros(1000, device="cuda").as_strided((9, 64), (32, 1)))),
                 lambda: ops.residual_norm(h, pre_norm=ops.Norm(), out=(None, "x"))]:
        with pytest.raises(ValueError):
            call()
    assert bool((windows == 0).all())
