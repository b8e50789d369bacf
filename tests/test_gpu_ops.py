"""Rotary positions, differential attention and the residual norms against their definitions in 64 bits.

Tolerances are bounds, not measurements.  A rounding to type t is off by at most u_t = eps / 2 of the value.  With e = 2^-24:
  rotary          angle: a fraction of a turn in fp32 (2^-25 turns = 1.9e-7 rad), sin / cos within 2 ulp, three roundings: 5e-7 (|u| + |w|) amplitude
  diff_attention  scores: d products summed in fp32; a weight's relative error is that of its exponent's argument; the 16-bit types round every weight to
                  the type before the product with v; the error of o is then at most the weights' relative error times A = P1 |v| + |lambda| P2 |v|
  residual_norm   sums of at most 64 dependent steps in fp32, then a handful of roundings
"""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {t: torch.finfo(t).eps / 2 for t in TYPES}
E = 2.0 ** -24
IDS = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    from radzero_amd import ops
    return ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def close(got, ref, tol, what=""):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound; worst {float((off / tol.clamp_min(1e-300))[bad].max())} x, first at {bad.nonzero()[0].tolist()}"


# ---- rotary -------------------------------------------------------------------------------------------------------------------

def rotary_ref(x, positions, freqs, layout, amplitude):
    """(reference, bound): positions (batch, tokens, axes), freqs (axes, pairs per axis) float64."""
    axes, per = freqs.shape
    angle = (positions.double()[..., None] * freqs).flatten(-2)[:, :, None]
    cos, sin = amplitude * angle.cos(), amplitude * angle.sin()
    P, X = axes * per, x.double()
    u, w = (X[..., :P], X[..., P:2 * P]) if layout == "half" else (X[..., 0:2 * P:2], X[..., 1:2 * P:2])
    a, b, m = u * cos - w * sin, u * sin + w * cos, 5e-7 * amplitude * (u.abs() + w.abs())
    join = (lambda y, z: torch.cat([y, z], -1)) if layout == "half" else (lambda y, z: torch.stack([y, z], -1).flatten(-2))
    rest = X[..., 2 * P:]
    ref = torch.cat([join(a, b), rest], -1)
    tol = torch.cat([join(m, m), torch.zeros_like(rest)], -1)
    tol[..., :2 * P] += U[x.dtype] * (ref[..., :2 * P].abs() + tol[..., :2 * P]) + (2.0 ** -25 if x.dtype == torch.float16 else 0)     # f16's smallest step
    return ref, tol


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("case", [  # batch, tokens, q heads, k heads, head_dim, rotary_dim, axes, far
    (1, 1, 1, 0, 2, 2, 1, 10), (8, 1, 16, 4, 128, 128, 1, 1 << 20), (2, 257, 12, 12, 64, 64, 2, 37), (3, 33, 6, 2, 96, 48, 1, 1 << 24), (1, 5, 2, 2, 80, 80, 2, 100),
    (2, 19, 3, 1, 7, 6, 1, 1000), (2, 6, 3, 3, 30, 18, 3, 50), (1, 3, 2, 1, 1024, 1024, 1, 100), (1, 1370, 12, 0, 64, 32, 1, 5000), (2, 9, 4, 4, 40, 24, 1, 64)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary(ops, dtype, case, layout):
    b, n, hq, hk, d, rot, axes, far = case
    g = gen(b * 1000 + n * 7 + d + rot)
    q, k = randn(g, b, n, hq, d, dtype=dtype), randn(g, b, n, hk, d, dtype=dtype) if hk else None
    pos = torch.randint(-far, far, (b, n, axes), generator=g, device="cuda")
    freqs, amplitude = ops.rotary_frequencies(rot, axes=axes, scaling={"kind": "yarn", "factor": 4, "original_length": 64}, device="cuda")
    table = freqs if axes > 1 else freqs[None]
    got = ops.rotary(q, k, positions=pos if axes > 1 else pos[..., 0], freqs=freqs, layout=layout, amplitude=amplitude)
    for x, y in zip((q, k), got if hk else (got, None)):
        if x is not None:
            close(y, *rotary_ref(x, pos, table, layout, amplitude), "rotary")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("case", [(2, 19, 3, 1, 70, 70, 1, 1000), (3, 40, 2, 2, 46, 28, 1, 1000), (1, 9, 5, 1, 12, 12, 3, 30), (1, 300, 4, 4, 26, 20, 1, 500)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_of_pairs(ops, dtype, case, layout):
    """Widths that divide by two and no further."""
    test_rotary(ops, dtype, case, layout)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_views_shared_positions_and_in_place(ops, dtype, layout):
    """q and k as views of one packed projection, heads before tokens, an odd offset, positions shared by the batch, outputs in place: the same bits, and nothing else written."""
    g = gen(3)
    b, n, h, d = 2, 21, 4, 64
    freqs, _ = ops.rotary_frequencies(48, device="cuda")
    pos = torch.arange(n, device="cuda") * 3
    packed = randn(g, b, n, 3 * h, d, dtype=dtype)
    q, k = packed[:, :, :h], packed[:, :, h:2 * h]
    want = ops.rotary(q.contiguous(), k.contiguous(), positions=pos.expand(b, n).contiguous(), freqs=freqs, layout=layout)
    close(want[0], *rotary_ref(q, pos.expand(b, n)[..., None], freqs[None], layout, 1.0))
    got = ops.rotary(q, k, positions=pos, freqs=freqs, layout=layout)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.rotary(heads_first, positions=pos, freqs=freqs, layout=layout), want[0])
    off = torch.zeros(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(b, n, h, d).copy_(q)          # not 16-byte aligned
    assert torch.equal(ops.rotary(off, positions=pos, freqs=freqs, layout=layout), want[0])
    v = packed[:, :, 2 * h:].clone()
    ops.rotary(q, k, positions=pos, freqs=freqs, layout=layout, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(packed[:, :, 2 * h:], v)


def test_rotary_far_positions_turn_back(ops):
    """Positions up to 2^31: turning by p and then by -p gives the input back."""
    g = gen(4)
    q = randn(g, 1, 64, 2, 64)
    pos = torch.randint(0, 2 ** 31 - 1, (1, 64), generator=g, device="cuda")
    freqs, _ = ops.rotary_frequencies(64, device="cuda")
    back = ops.rotary(ops.rotary(q, positions=pos, freqs=freqs), positions=-pos, freqs=freqs)
    # each direction: 5e-7, and the 64-bit angle's own 2^31 * 3 * 2^-53
    assert float((back - q).abs().max()) <= 2 * (5e-7 + 8e-7) * 2 * float(q.abs().max())


# ---- differential attention ----------------------------------------------------------------------------------------------------

def seen_keys(b, n_q, n_k, causal, lens, mask):
    """(batch, n_q, n_k) bool, from the definition."""
    j, i = torch.arange(n_k, device="cuda")[None, None], torch.arange(n_q, device="cuda")[None, :, None]
    n = (torch.full((b,), n_k, device="cuda") if lens is None else lens.long().clamp(0, n_k))[:, None, None]
    s = (j < n).expand(b, n_q, n_k)
    if mask is not None:
        s = s & (mask != 0)[:, None]
    if causal == "start":
        s = s & (j <= i)
    elif causal == "end":
        s = s & (j <= i + n - n_q)
    return s


def attention_ref(q, k, v, lam_qk, lambda_init, scale=None, causal=None, lens=None, mask=None, norm=None, eps=1e-5, out_scale=1.0):
    """(reference, bound) in float64, head by head."""
    b, n_q, h, w = q.shape
    n_k, hk, d = k.shape[1], k.shape[2], w // 2
    scale = d ** -0.5 if scale is None else scale
    seen = seen_keys(b, n_q, n_k, causal, lens, mask)
    any_seen = seen.any(-1, keepdim=True)
    u = U[q.dtype]
    ref = torch.zeros(b, n_q, h, w, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(ref)
    used = seen.any(1)[..., None]                        # (batch, n_k, 1): a key that nobody sees may hold anything
    for i in range(h):
        kv = i // (h // hk)
        lq = (lam_qk if lam_qk.dim() == 2 else lam_qk[i]).double()
        lam = float((lq[0] * lq[1]).sum().exp() - (lq[2] * lq[3]).sum().exp() + lambda_init)
        V = torch.where(used, v[:, :, kv].double(), 0.0)
        A = torch.zeros(b, n_q, w, dtype=torch.float64, device="cuda")
        o = torch.zeros_like(A)
        for m in range(2):
            Q, K = q[:, :, i, m * d:(m + 1) * d].double(), torch.where(used, k[:, :, kv, m * d:(m + 1) * d].double(), 0.0)
            s = (Q @ K.transpose(1, 2).contiguous()) * scale
            s = torch.where(seen, s, -math.inf)
            p = torch.where(any_seen, torch.softmax(torch.where(any_seen, s, 0.0), -1), 0.0)
            mag = torch.where(seen, (Q.abs() @ K.abs().transpose(1, 2).contiguous()) * scale, 0.0).amax(-1, keepdim=True)   # sum |q k| of the largest
            spread = 2 * mag
            # the score's d products (twice: it stands in the weight and in the sum), the exponent's argument, exp2 itself, the sums over the keys (a tree of partial sums: 64 + log)
            rel = E * (2 * d * mag + 2 * spread + 64 + n_k / 32) + (u if q.dtype != torch.float32 else 0)
            c = 1.0 if m == 0 else -lam
            o += c * (p @ V)
            A += abs(c) * rel * (p @ V.abs())
        # lambda itself: a dot of d products and two exps in fp32
        A += E * (2 * d + 16) * (p @ V.abs()) * float((lq[0] * lq[1]).sum().exp() + (lq[2] * lq[3]).sum().exp() + abs(lambda_init))
        if norm is not None:
            R = (o.square().mean(-1, keepdim=True) + eps).sqrt()
            t = A.square().mean(-1, keepdim=True).sqrt() / R
            f = out_scale * norm.double()
            y = f * o / R
            A = 1.1 * f.abs() * (A / R + (o.abs() / R) * t) + E * 16 * y.abs()
        else:
            y = out_scale * o
            A = abs(out_scale) * A + E * 4 * y.abs()
        ref[:, :, i], tol[:, :, i] = y, A
    tol += u * (ref.abs() + tol) + (2.0 ** -25 if q.dtype == torch.float16 else 1e-37)
    return ref, tol


def attention_inputs(seed, b, n_q, n_k, h, hk, d, dtype, std=1.5):
    g = gen(seed)
    q, k = randn(g, b, n_q, h, 2 * d, std=std, dtype=dtype), randn(g, b, n_k, hk, 2 * d, dtype=dtype)
    v = (randn(g, b, n_k, hk, 2 * d) + 0.5 * randn(g, hk, 2 * d)).to(dtype)
    return q, k, v, randn(g, 4, d, std=0.1), 1 + randn(g, 2 * d, std=0.1)


SHAPES = [  # batch, n_q, n_k, heads, kv_heads
    (1, 1, 1, 1, 1), (1, 1, 257, 6, 6), (2, 1, 63, 4, 2), (3, 5, 64, 4, 1), (2, 33, 65, 2, 2), (1, 64, 31, 3, 3), (2, 129, 200, 2, 1), (1, 257, 257, 6, 6), (1, 7, 1000, 8, 2),
    (1, 3, 5000, 6, 1), (2, 193, 700, 2, 2), (1, 31, 33, 12, 4), (1, 1, 9000, 2, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_diff_attention(ops, dtype, d, shape):
    q, k, v, lam, w = attention_inputs(sum(shape) + d, *shape, d, dtype)
    got = ops.diff_attention(q, k, v, lam, lambda_init=0.4)
    close(got, *attention_ref(q, k, v, lam, 0.4), "no norm")
    got = ops.diff_attention(q, k, v, lam, lambda_init=0.4, norm_weight=w, out_scale=0.6)
    close(got, *attention_ref(q, k, v, lam, 0.4, norm=w, out_scale=0.6), "norm")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(2, 1370, 1370, 2, 2), (1, 515, 2300, 4, 2), (4, 2, 20000, 4, 1), (33, 1, 700, 4, 4)], ids=str)
def test_diff_attention_longer(ops, dtype, shape):
    q, k, v, lam, w = attention_inputs(sum(shape), *shape, 64, dtype)
    got = ops.diff_attention(q, k, v, lam, lambda_init=0.4, norm_weight=w)
    close(got, *attention_ref(q, k, v, lam, 0.4, norm=w))
    assert torch.equal(got, ops.diff_attention(q, k, v, lam, lambda_init=0.4, norm_weight=w)), "two calls differ"


@pytest.mark.parametrize("d", [32, 64, 128])
def test_diff_attention_fp32_over_many_keys(ops, d):
    """The root mean square error of fp32 over 3500 keys.  32 keys' products join O at a time, n_k / 32 roundings of at most half a step at O's size, which go either way:
    sqrt(n_k / 32) of them; as much again for the weights and their sums."""
    q, k, v, lam, _ = attention_inputs(23, 1, 300, 3500, 4, 2, d, torch.float32, std=1.0)
    got = ops.diff_attention(q, k, v, lam, lambda_init=0.3).double()
    ref, _ = attention_ref(q, k, v, lam, 0.3)
    assert float((got - ref).square().sum().sqrt() / ref.square().sum().sqrt()) <= math.sqrt(2) * math.sqrt(3500 / 32) * E


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("causal", [None, "start", "end"])
@pytest.mark.parametrize("keys", ["all", "lens", "mask", "both"])
@pytest.mark.parametrize("shape", [(5, 70, 70, 4, 2), (5, 3, 301, 6, 1), (5, 140, 90, 2, 2), (5, 1, 4500, 2, 1)], ids=str)
def test_diff_attention_hidden_keys(ops, dtype, causal, keys, shape):
    """Lengths (zero, negative, one, beyond n_k), masks with empty rows and empty tiles, both causal alignments; NaN and infinities under every hidden key."""
    b, n_q, n_k, h, hk = shape
    q, k, v, lam, w = attention_inputs(n_q + n_k, *shape, 64, dtype)
    lens = torch.tensor([0, -3, 1, n_k + 5, n_k // 2 + 1], dtype=torch.int32, device="cuda") if keys in ("lens", "both") else None
    mask = None
    if keys in ("mask", "both"):
        mask = (torch.rand(b, n_k, generator=gen(9), device="cuda") < 0.7).long()
        mask[0] = 0
        mask[3, :n_k // 2] = 0
        mask[4, n_k // 3:] = 0
    used = seen_keys(b, n_q, n_k, causal, lens, mask).any(1)
    bad = torch.where(torch.arange(n_k, device="cuda") % 2 == 0, math.nan, math.inf)[None, :, None, None].to(dtype)
    k, v = torch.where(used[..., None, None], k, bad), torch.where(used[..., None, None], v, -bad)
    for norm in (None, w):
        got = ops.diff_attention(q, k, v, lam, lambda_init=0.3, causal=causal, kv_lens=lens, attention_mask=mask, norm_weight=norm)
        ref, tol = attention_ref(q, k, v, lam, 0.3, causal=causal, lens=lens, mask=mask, norm=norm)
        close(got, ref, tol)
        blind = ~seen_keys(b, n_q, n_k, causal, lens, mask).any(-1)
        assert bool((got[blind] == 0).all()), "a query that sees no key gets zeros"


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(9, 1, 6000, 4, 2), (9, 65, 5000, 2, 1), (64, 2, 900, 2, 2), (65, 2, 900, 2, 2), (1, 1, 40000, 1, 1), (2, 1, 300000, 1, 1)], ids=str)
def test_diff_attention_very_unequal_lengths(ops, dtype, shape):
    """Lengths that share the pieces of the key axis unequally: one long sequence among short, empty and negative ones, all empty, one sequence alone."""
    b, n_q, n_k, h, hk = shape
    q, k, v, lam, w = attention_inputs(sum(shape), *shape, 32, dtype)
    one_long = torch.tensor([0, 1, n_k, -7, 63, 64, 65, n_k // 2, 5], dtype=torch.int32, device="cuda").repeat(8)[:b].contiguous()
    for lens in (one_long, one_long.flip(0).contiguous(), torch.full_like(one_long, n_k), torch.zeros_like(one_long)):
        for causal in (None, "end"):
            got = ops.diff_attention(q, k, v, lam, lambda_init=0.3, causal=causal, kv_lens=lens, norm_weight=w)
            close(got, *attention_ref(q, k, v, lam, 0.3, causal=causal, lens=lens, norm=w))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("shape", [(1, 5, 1), (2, 4, 1), (3, 4, 2), (8, 2, 2), (7, 1, 1), (3, 1, 1), (1, 4, 2)], ids=str)
def test_diff_attention_few_rows(ops, dtype, d, shape):
    """One to eight query rows of a key head, the last block of them not full: causal edges inside a block, lengths, holes, and NaN under every hidden key."""
    n_q, h, hk = shape
    b, n_k = 4, 777
    q, k, v, lam, w = attention_inputs(n_q * 100 + h + d, b, n_q, n_k, h, hk, d, dtype)
    lens = torch.tensor([n_k, n_q + 1, 0, 500], dtype=torch.int32, device="cuda")
    mask = (torch.rand(b, n_k, generator=gen(5), device="cuda") < 0.6).long()
    for causal in (None, "start", "end"):
        for m in (None, mask):
            used = seen_keys(b, n_q, n_k, causal, lens, m).any(1)[..., None, None]
            bad_k, bad_v = torch.where(used, k, math.nan), torch.where(used, v, math.inf)
            got = ops.diff_attention(q, bad_k.to(dtype), bad_v.to(dtype), lam, lambda_init=0.3, causal=causal, kv_lens=lens, attention_mask=m, norm_weight=w)
            close(got, *attention_ref(q, k, v, lam, 0.3, causal=causal, lens=lens, mask=m, norm=w))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("causal", ["start", "end"])
def test_diff_attention_causal_over_several_rounds(ops, dtype, causal):
    """More blocks of query rows than the chip holds at a time, each row written once whatever the order they run in."""
    b, n, h, hk = 9, 700, 12, 6
    q, k, v, lam, w = attention_inputs(17, b, n, n, h, hk, 32, dtype)
    lens = torch.tensor([n, 1, n // 2, 0, n, 650, 33, n, n], dtype=torch.int32, device="cuda")
    got = ops.diff_attention(q, k, v, lam, lambda_init=0.3, causal=causal, kv_lens=lens, norm_weight=w, out=torch.full_like(q, 9.0))
    close(got, *attention_ref(q, k, v, lam, 0.3, causal=causal, lens=lens, norm=w))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_diff_attention_causal_rows_do_not_read_the_future(ops, dtype):
    """A NaN or infinity in a later token reaches that token's and later rows alone, whichever of k and v holds it."""
    b, n, h = 1, 150, 2
    q, k, v, lam, w = attention_inputs(11, b, n, n, h, h, 64, dtype)
    clean = ops.diff_attention(q, k, v, lam, lambda_init=0.3, causal="start", norm_weight=w)
    for at in (1, 40, 63, 64, 149):
        for x, value in ((k, math.nan), (v, math.nan), (v, math.inf), (k, math.inf)):
            held = x[0, at, :, 3].clone()
            x[0, at, :, 3] = value
            got = ops.diff_attention(q, k, v, lam, lambda_init=0.3, causal="start", norm_weight=w)
            x[0, at, :, 3] = held
            assert torch.equal(got[:, :at], clean[:, :at]), (at, value)
            if x is v or value != value:
                assert not bool(torch.isfinite(got[0, at:].float()).all(-1).any()), (at, value)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_diff_attention_large_scores(ops, dtype):
    """Scores of +-300 in both maps, maxima that grow along the keys, and a scale of the caller's."""
    b, n_q, n_k, h = 1, 40, 600, 2
    q, k, v, lam, w = attention_inputs(5, b, n_q, n_k, h, h, 64, dtype)
    k = (k.float() * torch.linspace(0.1, 6.0, n_k, device="cuda")[None, :, None, None]).to(dtype)
    got = ops.diff_attention(q, k, v, lam, lambda_init=0.3, scale=0.9)
    close(got, *attention_ref(q, k, v, lam, 0.3, scale=0.9))
    q[0, 3] = 0                                          # a row of equal scores
    q[0, 4] *= 1e-3
    got = ops.diff_attention(q, k, v, lam, lambda_init=0.3, scale=0.9, norm_weight=w)
    close(got, *attention_ref(q, k, v, lam, 0.3, scale=0.9, norm=w))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_diff_attention_views_and_neighbours(ops, dtype):
    """Packed projections, heads before tokens, per-head lambdas, a bool mask with strides, int64 lengths, an output inside a larger tensor whose other rows stay as they were."""
    b, n, h, hk, d = 3, 77, 4, 2, 32
    g = gen(21)
    packed = randn(g, b, n, h + 2 * hk, 2 * d, dtype=dtype)
    q, k, v = packed[:, :, :h], packed[:, :, h:h + hk], packed[:, :, h + hk:]
    lam = randn(g, h, 4, d, std=0.2)
    mask = (torch.rand(n, b, generator=g, device="cuda") < 0.8).t()
    lens = torch.tensor([n, 5, 1 << 40], device="cuda")
    ref, tol = attention_ref(q, k, v, lam, 0.2, causal="start", lens=lens, mask=mask)
    big = torch.full((b, n + 3, h + 1, 2 * d), 7.0, dtype=dtype, device="cuda")
    out = big[:, 1:n + 1, :h]
    got = ops.diff_attention(q, k, v, lam, lambda_init=0.2, causal="start", kv_lens=lens, attention_mask=mask, out=out)
    assert got is out
    close(out, ref, tol)
    assert bool((big[:, 0] == 7).all() and (big[:, n + 1:] == 7).all() and (big[:, :, h] == 7).all())
    qt, kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))
    assert torch.equal(ops.diff_attention(qt, kt, vt, lam, lambda_init=0.2, causal="start", kv_lens=lens, attention_mask=mask), out)


def test_diff_attention_of_no_keys_and_no_queries(ops):
    lam = torch.zeros(4, 32, device="cuda")
    q, k = torch.ones(2, 3, 4, 64, device="cuda"), torch.ones(2, 0, 2, 64, device="cuda")
    got = ops.diff_attention(q, k, k, lam, lambda_init=0.2, norm_weight=torch.ones(64, device="cuda"), out=torch.full_like(q, 5.0))
    assert bool((got == 0).all())
    many = torch.ones(2, 300, 4, 64, device="cuda")
    assert bool((ops.diff_attention(many, k, k, lam, lambda_init=0.2, out=torch.full_like(many, 5.0)) == 0).all())
    assert ops.diff_attention(q[:, :0], q, q, lam, lambda_init=0.2).shape == (2, 0, 4, 64)
    assert ops.diff_attention(q[:0], q[:0], q[:0], lam, lambda_init=0.2).shape == (0, 3, 4, 64)


def test_diff_attention_offsets_beyond_32_bits(ops):
    """A cache whose last rows lie more than 2^32 elements behind its first."""
    n_k, hk, d, step = 600, 1, 64, 1 << 23
    cache = torch.empty(step * n_k, dtype=torch.bfloat16, device="cuda")
    q, k, v, lam, w = attention_inputs(8, 1, 2, n_k, 4, hk, d, torch.bfloat16)
    far = [cache.as_strided((1, n_k, hk, 2 * d), (0, step, 2 * d, 1), o) for o in (0, 2 * d)]
    assert step * (n_k - 1) > 1 << 32
    far[0].copy_(k), far[1].copy_(v)
    assert torch.equal(ops.diff_attention(q, *far, lam, lambda_init=0.3, norm_weight=w), ops.diff_attention(q, k, v, lam, lambda_init=0.3, norm_weight=w))


def test_diff_attention_tokens_far_apart(ops):
    """A cache whose tokens lie 0.7 GB apart: the offsets within one copy of a few tokens pass 32 bits too."""
    n_k, d, step = 64, 32, 5 << 26
    cache = torch.empty(step * n_k, dtype=torch.bfloat16, device="cuda")
    for n_q in (1, 8, 40):
        q, k, v, lam, w = attention_inputs(9, 1, n_q, n_k, 1, 1, d, torch.bfloat16)
        far = [cache.as_strided((1, n_k, 1, 2 * d), (0, step, 2 * d, 1), o) for o in (0, 2 * d)]
        far[0].copy_(k), far[1].copy_(v)
        assert torch.equal(ops.diff_attention(q, *far, lam, lambda_init=0.3, norm_weight=w), ops.diff_attention(q, k, v, lam, lambda_init=0.3, norm_weight=w)), n_q
    del cache, far
    torch.cuda.empty_cache()


def test_more_rows_than_one_launch_takes(ops):
    g = gen(41)
    n = (1 << 23) + 13
    q, pos = randn(g, 1, n, 1, 2, dtype=torch.bfloat16), torch.randint(0, 1000, (n,), generator=g, device="cuda")
    freqs = torch.tensor([0.25], dtype=torch.float64, device="cuda")
    got = ops.rotary(q, positions=pos, freqs=freqs)
    for at in (slice(0, 4096), slice(n - 4096, n)):
        assert torch.equal(got[:, at], ops.rotary(q[:, at], positions=pos[at], freqs=freqs))
    residual = randn(g, n, 3)
    pre = ops.Norm(kind="rms")
    x = ops.residual_norm(residual, pre_norm=pre)[1]
    for at in (slice(0, 4096), slice((1 << 22) - 50, (1 << 22) + 50), slice(n - 4096, n)):
        assert torch.equal(x[at], ops.residual_norm(residual[at], pre_norm=pre)[1])


# ---- residual norms ------------------------------------------------------------------------------------------------------------

def norm_ref(x, ex, kind, weight, bias, eps):
    """(norm of x, bound) given x's own bound ex: sums of at most 64 dependent fp32 steps."""
    K = 64 * E
    if kind == "layer":
        ec = ex + ex.mean(-1, keepdim=True) + K * x.abs().mean(-1, keepdim=True) + E * x.abs()
        x = x - x.mean(-1, keepdim=True)
    else:
        ec = ex
    sigma = (x.square().mean(-1, keepdim=True) + eps).sqrt()
    z = x / sigma
    t = ec.square().mean(-1, keepdim=True).sqrt() / sigma
    ez = 1.05 * (ec / sigma + z.abs() * (t + K))
    w = 1.0 if weight is None else weight.double()
    b = 0.0 if bias is None else bias.double()
    y = z * w + b
    return y, ez * abs(w) + 4 * E * ((z * w).abs() + y.abs())


def residual_ref(residual, y, pre, post, scale, gate, alpha):
    r, er = residual.double() * alpha, E * (residual.double() * alpha).abs()
    if y is not None:
        t, et = y.double(), torch.zeros_like(r)
        if post is not None:
            t, et = norm_ref(t, et, post.kind, post.weight, post.bias, post.eps)
        f = torch.ones((), dtype=torch.float64, device="cuda") if scale is None else scale.double()
        f = f if gate is None else f * gate.double()
        er = er + f.abs() * et + 4 * E * (f * t).abs()
        r = r + f * t
        er = er + E * r.abs()
    tiny = 2.0 ** -25
    out = (r, er + U[residual.dtype] * (r.abs() + er) + (tiny if residual.dtype == torch.float16 else 0))
    if pre is None:
        return out, None
    x, ex = norm_ref(r, er, pre.kind, pre.weight, pre.bias, pre.eps)
    return out, (x, ex)


def finish(x, ex, dtype):
    return x, ex + U[dtype] * (x.abs() + ex) + (2.0 ** -25 if dtype == torch.float16 else 1e-37)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 5), (1, 5, 64), (3, 7, 255), (2, 9, 768), (1, 3, 1001), (2, 4, 1024), (1, 3, 1027), (1, 2, 2049), (2, 2, 4096), (1, 3, 7777), (1, 2, 16384), (2, 513, 768)],
                         ids=str)
def test_residual_norm(ops, dtype, kind, shape):
    b, n, d = shape
    g = gen(b + n + d)
    y = randn(g, b, n, d, dtype=dtype)
    pre = ops.Norm(1 + randn(g, d, std=0.1), randn(g, d, std=0.1) if kind == "layer" else None, 1e-6, kind)
    post = ops.Norm(1 + randn(g, d, std=0.1), None, 1e-5, kind)
    scale, gate = randn(g, d, std=0.3), randn(g, b, d, std=0.5)
    for rt in {torch.float32, dtype}:
        residual = (randn(g, b, n, d, std=2.0) + 1.5).to(rt)
        for po, sc, ga, alpha in ((None, None, None, 1.0), (post, scale, None, 1.0), (None, scale, gate, 0.7), (post, None, gate[:, None].expand(b, n, d).contiguous(), 1.0), (post, scale, gate[0], -1.3)):
            r, x = ops.residual_norm(residual, y, pre_norm=pre, post_norm=po, scale=sc, gate=ga, alpha=alpha)
            full = ga if ga is None or ga.dim() != 2 else ga[:, None]
            out, norm = residual_ref(residual, y, pre, po, sc, full, alpha)
            assert r.dtype == rt and x.dtype == dtype
            close(r, *out, "r")
            close(x, *finish(*norm, dtype), "x")
        r, x = ops.residual_norm(residual, pre_norm=pre, dtype=dtype)
        assert r is residual
        close(x, *finish(*residual_ref(residual, None, pre, None, None, None, 1.0)[1], dtype), "pre-norm alone")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_residual_norm_views_in_place_and_neighbours(ops, dtype):
    """Rows that are slices (the patches without their first token), odd strides, in place: the same bits, the other rows untouched."""
    g = gen(31)
    b, n, d = 3, 10, 771
    big, by = randn(g, b, n + 1, d + 2), randn(g, b, n + 1, d + 1, dtype=dtype)
    h, y = big[:, 1:, :d], by[:, 1:, 1:]
    pre, post, scale = ops.Norm(1 + randn(g, d, std=0.1), randn(g, d, std=0.1)), ops.Norm(kind="rms"), randn(g, d)
    want = ops.residual_norm(h.contiguous(), y.contiguous(), pre_norm=pre, post_norm=post, scale=scale)
    got = ops.residual_norm(h, y, pre_norm=pre, post_norm=post, scale=scale)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    keep_h, keep_y = big.clone(), by.clone()
    r, x = ops.residual_norm(h, y, pre_norm=pre, post_norm=post, scale=scale, out=(h, y))
    assert r is h and x is y and torch.equal(h, want[0]) and torch.equal(y, want[1])
    assert torch.equal(big[:, 0], keep_h[:, 0]) and torch.equal(big[:, :, d:], keep_h[:, :, d:]) and torch.equal(by[:, 0], keep_y[:, 0]) and torch.equal(by[:, :, 0], keep_y[:, :, 0])
    two = ops.residual_norm(want[0][0], want[1][0], pre_norm=None, gate=randn(g, n, d))
    assert two[1] is None and two[0].shape == (n, d)
    r, x = ops.residual_norm(h[:, :0], y[:, :0], pre_norm=pre)
    assert r.shape == (b, 0, d) and x.shape == (b, 0, d)


@pytest.mark.parametrize("d", [1, 3, 16, 17, 64, 65, 128, 129, 190, 193, 256, 257, 385, 512, 513, 768, 769, 1024, 1025], ids=str)
def test_residual_norm_many_rows(ops, d):
    """More rows than waves, so that a wave takes several, with runs that cross from one sample to the next: each sample's own gate, a gate per row, in place."""
    g = gen(35 + d)
    b, n = 5, 2741
    residual, y = randn(g, b, n, d), randn(g, b, n, d, dtype=torch.bfloat16)
    pre, post, scale = ops.Norm(1 + randn(g, d, std=0.1), randn(g, d, std=0.1)), ops.Norm(1 + randn(g, d, std=0.1), kind="rms"), randn(g, d, std=0.3)
    per_sample = randn(g, b, d, std=0.5)
    for gate in (None, per_sample, randn(g, b, n, d, std=0.5)):
        want, norm = residual_ref(residual, y, pre, post, scale, per_sample[:, None] if gate is per_sample else gate, 1.0)
        r, x = ops.residual_norm(residual, y, pre_norm=pre, post_norm=post, scale=scale, gate=gate)
        close(r, *want, "r")
        close(x, *finish(*norm, torch.bfloat16), "x")
    h = residual.clone()
    again = ops.residual_norm(h, y, pre_norm=pre, post_norm=post, scale=scale, gate=gate, out=(h, None))
    assert again[0] is h and torch.equal(h, r) and torch.equal(again[1], x)


def test_residual_norm_keeps_a_large_mean(ops):
    """A row whose mean is 4000 times its spread: a sum of squares minus a squared mean would have nothing left."""
    g = gen(33)
    residual = randn(g, 4, 768) + 4000.0
    _, x = ops.residual_norm(residual, pre_norm=ops.Norm())
    close(x, *finish(*residual_ref(residual, None, ops.Norm(), None, None, None, 1.0)[1], torch.float32))


# ---- refusals, streams, graphs, the block ---------------------------------------------------------------------------------------

def test_operators_refuse(ops):
    q = torch.zeros(2, 4, 4, 64, device="cuda", dtype=torch.bfloat16)
    lam, freqs, pos = torch.zeros(4, 32, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda"), torch.arange(4, device="cuda")
    bad = [
        lambda: ops.rotary(q, q[:, :3], positions=pos, freqs=freqs), lambda: ops.rotary(q, q.float(), positions=pos, freqs=freqs),
        lambda: ops.rotary(q, positions=pos.int(), freqs=freqs), lambda: ops.rotary(q, positions=pos[:3], freqs=freqs), lambda: ops.rotary(q, positions=pos, freqs=freqs.float()),
        lambda: ops.rotary(q, positions=pos, freqs=torch.ones(33, dtype=torch.float64, device="cuda")), lambda: ops.rotary(q, positions=pos, freqs=freqs, layout="thirds"),
        lambda: ops.rotary(q, positions=pos, freqs=freqs.view(2, 16)), lambda: ops.rotary(q.transpose(2, 3), positions=pos, freqs=freqs),
        lambda: ops.rotary(q, positions=pos, freqs=freqs, out=q[:, :2]), lambda: ops.rotary(q.half().requires_grad_(), positions=pos, freqs=freqs),
        lambda: ops.rotary(q[:, :, :0], positions=pos, freqs=freqs), lambda: ops.rotary(q.cpu(), positions=pos, freqs=freqs), lambda: ops.rotary(q.double(), positions=pos, freqs=freqs),
        lambda: ops.diff_attention(q, q[:, :, :3], q[:, :, :3], lam, lambda_init=0.1), lambda: ops.diff_attention(q, q[:1], q[:1], lam, lambda_init=0.1),
        lambda: ops.diff_attention(q, q, q[:, :3], lam, lambda_init=0.1), lambda: ops.diff_attention(q[..., :48], q[..., :48], q[..., :48], lam, lambda_init=0.1),
        lambda: ops.diff_attention(q, q, q, lam.half(), lambda_init=0.1), lambda: ops.diff_attention(q, q, q, lam[:3], lambda_init=0.1),
        lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.1, causal=True), lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.1, scale=-1.0),
        lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.1, kv_lens=torch.ones(3, dtype=torch.int32, device="cuda")),
        lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.1, kv_lens=torch.ones(2, device="cuda")),
        lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.1, attention_mask=torch.ones(2, 4, device="cuda")),
        lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.1, attention_mask=torch.ones(2, 5, dtype=torch.int64, device="cuda")),
        lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.1, norm_weight=torch.ones(32, device="cuda")),
        lambda: ops.diff_attention(q, q, q, lam, lambda_init=0.1, out=q[:, :1].expand(2, 4, 4, 64)),
        lambda: ops.diff_attention(torch.zeros(2 * 4 * 4 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, 4, 4, 64), q, q, lam, lambda_init=0.1),
        lambda: ops.diff_attention(q.float().requires_grad_(), q.float(), q.float(), lam, lambda_init=0.1),
        lambda: ops.residual_norm(q[0, 0].float(), q[0, 1, :3], pre_norm=ops.Norm()), lambda: ops.residual_norm(q[0, 0].half(), q[0, 1], pre_norm=ops.Norm()),
        lambda: ops.residual_norm(q[0, 0], q[0, 1], pre_norm=ops.Norm(kind="batch")), lambda: ops.residual_norm(q[0, 0], q[0, 1], pre_norm=ops.Norm(weight=torch.ones(65, device="cuda"))),
        lambda: ops.residual_norm(q[0, 0], scale=torch.ones(64, device="cuda"), pre_norm=None), lambda: ops.residual_norm(q[0, 0], q[0, 1], pre_norm=None, gate=torch.ones(3, 64, device="cuda")),
        lambda: ops.residual_norm(q, q, pre_norm=ops.Norm()), lambda: ops.residual_norm(q[0, 0], q[0, 1], pre_norm=ops.Norm(eps=-1.0)),
        lambda: ops.residual_norm(torch.zeros(2, 16385, device="cuda"), pre_norm=ops.Norm()), lambda: ops.residual_norm(q[0, 0], q[0, 1], pre_norm=None, out=(None, q[0, 1])),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError(f"call {i} was not refused")


def test_operators_on_a_side_stream_and_in_graphs(ops):
    """Two captured graphs that share nothing but their code, replayed in turn with eager calls between: every replay gives the eager call's bits for its inputs."""
    d, shapes = 64, [(2, 1, 9000, 4, 2), (1, 300, 300, 4, 4)]
    freqs, _ = ops.rotary_frequencies(2 * d, device="cuda")

    def step(s):
        q = ops.rotary(s["q"], positions=s["pos"], freqs=freqs)
        o = ops.diff_attention(q, s["k"], s["v"], s["lam"], lambda_init=0.3, causal="end", kv_lens=s["lens"], norm_weight=s["w"])
        return ops.residual_norm(s["h"], o.flatten(2), pre_norm=ops.Norm())

    def fill(s, seed):
        b, n_q, n_k, h, hk = s["shape"]
        q, k, v, _, _ = attention_inputs(seed, b, n_q, n_k, h, hk, d, torch.bfloat16)
        s["q"].copy_(q), s["k"].copy_(k), s["v"].copy_(v), s["h"].copy_(randn(gen(seed), *s["h"].shape))
        s["lens"].copy_(torch.randint(1, n_k + 1, (b,), generator=gen(seed), device="cuda"))

    made, side = [], torch.cuda.Stream()
    for shape in shapes:
        b, n_q, n_k, h, hk = shape
        q, k, v, lam, w = attention_inputs(1, *shape, d, torch.bfloat16)
        s = {"shape": shape, "q": q, "k": k, "v": v, "lam": lam, "w": w, "pos": torch.arange(n_q, device="cuda") + 7, "h": randn(gen(2), b, n_q, h * 2 * d),
             "lens": torch.full((b,), n_k, dtype=torch.int32, device="cuda")}
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(s)
        made.append((s, graph, out))
    for turn in range(4):
        for s, graph, out in made:
            fill(s, 100 + turn)
            graph.replay()
            torch.cuda.synchronize()
            want = step(s)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), (s["shape"], turn)
    s = made[0][0]
    want = step(s)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(s)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_a_differential_block(ops, dtype):
    """norm -> q|k|v product -> rotary -> differential attention -> output product -> gate, scale, residual and next norm, with the framework's own products: each operator
    against its definition on what the one before it gave."""
    from radzero_amd import _lib
    lib, code = _lib.load(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    b, n, h, d = 2, 128, 6, 64
    dim, g = h * 2 * d, gen(77)

    def product(x, w, bias):
        out = torch.empty(x.shape[0], w.shape[0], dtype=dtype, device="cuda")
        P = lambda t: ctypes.c_void_p(t.data_ptr())                          # noqa: E731
        _lib.check(lib.rz_gemm(code, 0, P(x), P(w), P(bias), P(out), x.shape[0], w.shape[0], x.shape[1], ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "rz_gemm")
        return out

    hid = randn(g, b, n, dim)
    w_qkv, w_o = randn(g, 3 * dim, dim, std=dim ** -0.5, dtype=dtype), randn(g, dim, dim, std=dim ** -0.5, dtype=dtype)
    b_qkv, b_o = randn(g, 3 * dim, std=0.1), randn(g, dim, std=0.1)
    pre, post, nxt = (ops.Norm(1 + randn(g, dim, std=0.1), randn(g, dim, std=0.1)) for _ in range(3))
    lam, sub, scale, gate = randn(g, 4, d, std=0.1), 1 + randn(g, 2 * d, std=0.1), randn(g, dim, std=0.1), randn(g, b, dim)
    grid = torch.stack(torch.meshgrid(torch.arange(8), torch.arange(16), indexing="ij"), -1).reshape(n, 2).cuda()
    freqs, _ = ops.rotary_frequencies(d, axes=2, device="cuda")

    _, x = ops.residual_norm(hid, pre_norm=pre, dtype=dtype)
    close(x, *finish(*residual_ref(hid, None, pre, None, None, None, 1.0)[1], dtype), "first norm")
    qkv = product(x.view(b * n, dim), w_qkv, b_qkv).view(b, n, 3 * h, 2 * d)
    q, k, v = qkv[:, :, :h], qkv[:, :, h:2 * h], qkv[:, :, 2 * h:]
    # each map's half of a head is turned by itself: (tokens, 2 heads, d) views of q and k
    half = lambda t: t.reshape(b, n, 2 * h, d) if t.is_contiguous() else t.as_strided((b, n, 2 * h, d), (t.stride(0), t.stride(1), d, 1), t.storage_offset())      # noqa: E731
    before = qkv.clone()
    ops.rotary(half(q), half(k), positions=grid, freqs=freqs, out=(half(q), half(k)))
    for t, was in ((q, before[:, :, :h]), (k, before[:, :, h:2 * h])):
        close(half(t), *rotary_ref(half(was), grid.expand(b, n, 2), freqs, "half", 1.0), "rotary")
    ctx = ops.diff_attention(q, k, v, lam, lambda_init=0.2, norm_weight=sub, out_scale=0.8)
    close(ctx, *attention_ref(q, k, v, lam, 0.2, norm=sub, out_scale=0.8), "attention")
    y = product(ctx.view(b * n, dim), w_o, b_o).view(b, n, dim)
    r, nx = ops.residual_norm(hid, y, pre_norm=nxt, post_norm=post, scale=scale, gate=gate)
    out, norm = residual_ref(hid, y, nxt, post, scale, gate[:, None], 1.0)
    close(r, *out, "residual")
    close(nx, *finish(*norm, dtype), "next norm")
