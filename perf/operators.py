"""The operators of a differential-attention encoder block, in their plain form and as calls of radzero_amd.ops.

Rotary positions, differential attention, and the block's norms with its gate and residual scale.  `listed()` names the
measured cases, `draw()` makes more of the same ranges, `prepare()` makes what a caller has in hand, `run()` is one pass.
"""
import math

import torch

own = False                     # False: the plain form in elementary torch operations; True: the framework's kernels

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _attention(name, dtype, batch, n_q, n_k, heads, kv_heads, dim, causal="no", keys="all", norm=True):
    # causal: "start" = query i is token i, "end" = the queries are the last tokens of their sequence
    # keys: "all" = every key counts, "lens" = a length per batch entry, "mask" = a padded 0/1 mask with holes
    # packed projections (q | k | v of one product) where queries and keys are the same tokens
    return {"name": name, "op": "diff_attention", "dtype": dtype, "batch": batch, "n_q": n_q, "n_k": n_k, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "causal": causal, "keys": keys, "norm": norm}


def _rotary(name, dtype, batch, tokens, q_heads, k_heads, dim, rotary_dim, axes, layout, far):
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "tokens": tokens, "q_heads": q_heads,
            "k_heads": k_heads, "dim": dim, "rotary_dim": rotary_dim, "axes": axes, "layout": layout, "far": far}


def _residual(name, dtype, batch, rows, dim, kind, post, gate, scale, resid):
    return {"name": name, "op": "residual_norm", "dtype": dtype, "batch": batch, "rows": rows, "dim": dim, "kind": kind,
            "post": post, "gate": gate, "scale": scale, "resid": resid}


def listed():
    return [
        # one prompt vector over the patches of one 224-pixel image: all latency
        _attention("attend_1_over_257", "bf16", 1, 1, 257, 6, 6, 64),
        # an encoder layer of a batch of 518-pixel images (1 + 37 * 37 tokens)
        _attention("encoder_518_bf16", "bf16", 8, 1370, 1370, 6, 6, 64),
        # an encoder layer at 1024 pixels (1 + 73 * 73 tokens): the largest
        _attention("encoder_1024_bf16", "bf16", 4, 5330, 5330, 6, 6, 64),
        # the 1e-3 mode's type, one 518-pixel image
        _attention("encoder_518_f32", "f32", 1, 1370, 1370, 6, 6, 64),
        # 193 prompts over the patches of images of several sizes, up to 1536 pixels (1 + 109 * 109 tokens)
        _attention("prompts_over_patches_f16", "f16", 4, 193, 11882, 6, 6, 64, keys="lens", norm=False),
        # a padded batch of report texts, causal, shared key heads
        _attention("causal_text_f16", "f16", 14, 512, 512, 12, 4, 32, causal="start", keys="mask"),
        # one new token per sequence over long caches of unequal lengths, shared key heads
        _attention("one_token_long_cache_bf16", "bf16", 8, 1, 32768, 16, 4, 64, causal="end", keys="lens"),
        # one new token's positions per sequence, far into a long text
        _rotary("rotary_one_token", "bf16", 8, 1, 16, 4, 128, 128, 1, "interleaved", 1 << 20),
        # row and column positions of the patches of a full batch at 1024 pixels
        _rotary("rotary_patches_1024", "bf16", 32, 5330, 12, 12, 64, 64, 2, "half", 73),
        # the norms of one token per sequence
        _residual("norm_8_rows", "bf16", 8, 1, 768, "layer", True, False, True, "f32"),
        # the norms between attention and MLP of a full batch at 1024 pixels
        _residual("norm_batch_1024", "bf16", 32, 5330, 768, "layer", True, False, True, "f32"),
        # a gated block with root-mean-square norms and an odd width
        _residual("norm_gated_odd_f16", "f16", 8, 1370, 1001, "rms", True, True, False, "f16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["diff_attention", "diff_attention", "diff_attention", "rotary", "residual_norm"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "diff_attention":
        dim = rng.choice([32, 64, 64, 128])
        kv_heads = rng.choice([1, 2, 3, 4, 6])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
        use = rng.choice(["encoder", "prompts", "text", "token"])
        causal, keys = "no", rng.choice(["all", "lens", "mask"])
        if use == "encoder":
            n_q = n_k = _log(rng, 17, 5330)
        elif use == "prompts":
            n_q, n_k = _log(rng, 1, 256), _log(rng, 64, 12000)
        elif use == "text":
            n_q = n_k = _log(rng, 1, 2048)
            causal = "start"
        else:
            n_q, n_k, causal = rng.choice([1, 1, 1, 2, 5]), _log(rng, 16, 65536), "end"
            n_k = max(n_k, n_q)
        most = 3e8 if dtype != "f32" else 3e7           # query-key pairs of all heads, as head dim 64
        batch = max(1, min(32, int(most / (heads * n_q * n_k * dim / 64))))
        batch = max(1, min(batch, int(6e8 / (n_k * kv_heads * dim * 4 * SIZE[dtype]))))
        batch = rng.randint(1, batch)
        c = _attention("", dtype, batch, n_q, n_k, heads, kv_heads, dim, causal, keys, rng.random() < 0.6)
    elif op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128])
        axes = rng.choice([1, 1, 2])
        rotary_dim = rng.choice([dim, dim, dim // 2])
        batch, tokens = rng.randint(1, 16), _log(rng, 1, 5330)
        q_heads = rng.choice([4, 6, 12, 16])
        c = _rotary("", dtype, batch, tokens, q_heads, rng.choice([0, q_heads // 2, q_heads]), dim, rotary_dim, axes,
                    rng.choice(["half", "interleaved"]), rng.choice([100, 10000, 1 << 20, 1 << 24]))
    else:
        dim = rng.choice([_log(rng, 1, 8192), 64 * _log(rng, 1, 128)])
        rows = max(1, min(_log(rng, 1, 100000), int(9e7 / dim)))
        batch = rng.randint(1, min(16, rows))
        c = _residual("", dtype, batch, max(1, rows // batch), dim, rng.choice(["layer", "rms"]), rng.random() < 0.6,
                      rng.random() < 0.5, rng.random() < 0.5, rng.choice(["f32", "f32", dtype]))
    del c["name"]
    return c


def _lens(c):
    """Keys of each batch entry: from all of them down to about half."""
    return [c["n_k"] - b * c["n_k"] // (2 * c["batch"]) for b in range(c["batch"])]


def _holes(c):
    """Every 7th key of a mask is a hole."""
    return [sum(1 for j in range(n) if j % 7 != 3) for n in _lens(c)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[c["dtype"]]

    def randn(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    if c["op"] == "diff_attention":
        b, n_q, n_k, h, hk, d = c["batch"], c["n_q"], c["n_k"], c["heads"], c["kv_heads"], c["dim"]
        mean = randn(hk, 2 * d, std=0.5)                # values have a mean per channel, as projections with a bias give them
        if n_q == n_k:                                  # q | k | v of one projection
            qkv = randn(b, n_q, h + 2 * hk, 2 * d, dtype=t)
            q, k, v = qkv[:, :, :h], qkv[:, :, h:h + hk], qkv[:, :, h + hk:]
        else:
            q, k, v = randn(b, n_q, h, 2 * d, dtype=t), randn(b, n_k, hk, 2 * d, dtype=t), randn(b, n_k, hk, 2 * d, dtype=t)
        q *= 1.5
        v += mean.to(t)
        s = {"op": c["op"], "q": q, "k": k, "v": v, "lambda_qk": randn(4, d, std=0.1), "lambda_init": 0.8 - 0.6 * math.exp(-0.9),
             "causal": c["causal"], "kv_lens": None, "mask": None, "norm": None}
        lens = torch.tensor(_lens(c), device="cuda", dtype=torch.int32).roll(seed % b)
        if c["keys"] == "lens":
            s["kv_lens"] = lens
        elif c["keys"] == "mask":
            j = torch.arange(n_k, device="cuda")
            s["mask"] = ((j[None] < lens[:, None]) & (j % 7 != 3)[None]).long()
        if c["norm"]:
            s["norm"] = 1 + randn(2 * d, std=0.1)
        return s
    if c["op"] == "rotary":
        b, n, d, a = c["batch"], c["tokens"], c["dim"], c["axes"]
        pairs = c["rotary_dim"] // (2 * a)
        freqs = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
        shape = (b, n) if a == 1 else (b, n, a)
        positions = torch.randint(0, c["far"], shape, generator=g, device="cuda")
        return {"op": c["op"], "q": randn(b, n, c["q_heads"], d, dtype=t), "k": randn(b, n, c["k_heads"], d, dtype=t) if c["k_heads"] else None,
                "positions": positions, "freqs": freqs if a == 1 else freqs.expand(a, pairs).contiguous(), "layout": c["layout"]}
    b, n, d = c["batch"], c["rows"], c["dim"]
    bias = c["kind"] == "layer"
    s = {"op": c["op"], "kind": c["kind"], "residual": randn(b, n, d, std=2.0, dtype=TYPES[c["resid"]]), "y": randn(b, n, d, dtype=t),
         "pre": (1 + randn(d, std=0.1), randn(d, std=0.1) if bias else None), "post": None, "gate": None, "scale": None}
    if c["post"]:
        s["post"] = (1 + randn(d, std=0.1), randn(d, std=0.1) if bias else None)
    if c["gate"]:
        s["gate"] = randn(b, d, std=0.5)
    if c["scale"]:
        s["scale"] = randn(d, std=0.2)
    return s


EPS_ATTENTION, EPS_NORM = 1e-5, 1e-6


def _plain_diff_attention(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, n_q, h, d = q.shape[0], q.shape[1], q.shape[2], q.shape[3] // 2
    n_k, hk = k.shape[1], k.shape[2]
    # (batch, kv head, heads of its group, map, rows, d) against (batch, kv head, 1, map, keys, d)
    q = q.view(b, n_q, hk, h // hk, 2, d).permute(0, 2, 3, 4, 1, 5)
    k = k.view(b, n_k, hk, 1, 2, d).permute(0, 2, 3, 4, 1, 5)
    x = torch.matmul(q.reshape(b, hk, -1, 2, n_q, d), k.transpose(-1, -2).contiguous()) / math.sqrt(d)
    lens = s["kv_lens"] if s["kv_lens"] is not None else torch.full((b,), n_k, device=q.device)
    j = torch.arange(n_k, device=q.device)
    seen = j[None, None] < lens[:, None, None]
    if s["mask"] is not None:
        seen = seen & (s["mask"] != 0)[:, None]
    if s["causal"] != "no":
        i = torch.arange(n_q, device=q.device)
        first = lens - n_q if s["causal"] == "end" else torch.zeros_like(lens)
        seen = seen & (j[None, None] <= i[None, :, None] + first[:, None, None])
    x = torch.where(seen[:, None, None, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    x = x / x.sum(-1, keepdim=True).clamp_min(1e-30)
    lq = s["lambda_qk"]
    lam = torch.exp((lq[0] * lq[1]).sum()) - torch.exp((lq[2] * lq[3]).sum()) + s["lambda_init"]
    o = torch.matmul(x[:, :, :, 0] - lam * x[:, :, :, 1], v.permute(0, 2, 1, 3)[:, :, None].contiguous())
    if s["norm"] is not None:
        o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS_ATTENTION) * s["norm"] * (1 - s["lambda_init"])
    return o.permute(0, 3, 1, 2, 4).reshape(b, n_q, h, 2 * d).to(s["q"].dtype)


def _plain_turn(x, cos, sin, layout):
    p = cos.shape[-1]
    r, rest = x[..., :2 * p].float(), x[..., 2 * p:]
    u, w = (r[..., :p], r[..., p:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    u, w = u * cos - w * sin, u * sin + w * cos
    r = torch.cat([u, w], -1) if layout == "half" else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([r.to(x.dtype), rest], -1)


def _plain_rotary(s):
    pos, freqs = s["positions"].double(), s["freqs"]
    angle = pos[..., None] * freqs if freqs.dim() == 1 else (pos[..., None] * freqs).flatten(-2)     # 64 bits: far positions
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    q = _plain_turn(s["q"], cos, sin, s["layout"])
    return [q] if s["k"] is None else [q, _plain_turn(s["k"], cos, sin, s["layout"])]


def _plain_norm(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS_NORM) * weight
    return x if bias is None else x + bias


def _plain_residual_norm(s):
    t = s["y"].float()
    if s["post"] is not None:
        t = _plain_norm(t, s["kind"], *s["post"])
    if s["scale"] is not None:
        t = t * s["scale"]
    if s["gate"] is not None:
        t = t * s["gate"][:, None]
    r = s["residual"].float() + t
    return [r.to(s["residual"].dtype), _plain_norm(r, s["kind"], *s["pre"]).to(s["y"].dtype)]


def run(state):
    s = state
    if own:
        from radzero_amd import ops
        if s["op"] == "diff_attention":
            norm = s["norm"]
            return ops.diff_attention(s["q"], s["k"], s["v"], s["lambda_qk"], lambda_init=s["lambda_init"], causal=None if s["causal"] == "no" else s["causal"], kv_lens=s["kv_lens"],
                                      attention_mask=s["mask"], norm_weight=norm, norm_eps=EPS_ATTENTION,
                                      out_scale=1.0 if norm is None else 1 - s["lambda_init"])
        if s["op"] == "rotary":
            got = ops.rotary(s["q"], s["k"], positions=s["positions"], freqs=s["freqs"], layout=s["layout"])
            return [got] if s["k"] is None else list(got)
        pre = ops.Norm(*s["pre"], eps=EPS_NORM, kind=s["kind"])
        post = None if s["post"] is None else ops.Norm(*s["post"], eps=EPS_NORM, kind=s["kind"])
        return list(ops.residual_norm(s["residual"], s["y"], pre_norm=pre, post_norm=post, scale=s["scale"], gate=s["gate"]))
    if s["op"] == "diff_attention":
        return _plain_diff_attention(s)
    return _plain_rotary(s) if s["op"] == "rotary" else _plain_residual_norm(s)


def work(case):
    c = case
    e = SIZE[c["dtype"]]
    if c["op"] == "diff_attention":
        lens = [c["n_k"]] * c["batch"] if c["keys"] == "all" else _lens(c) if c["keys"] == "lens" else _holes(c)
        keys = sum(lens)
        if c["causal"] != "no":
            # query i sees the keys up to its own token; the holes of a mask take the same share everywhere
            ends = [c["n_k"]] * c["batch"] if c["keys"] == "all" else _lens(c)
            first = [n - c["n_q"] if c["causal"] == "end" else 0 for n in (ends if c["keys"] == "lens" else [c["n_k"]] * c["batch"])]
            pairs = sum(sum(max(0, min(n, i + f + 1)) for i in range(c["n_q"])) * seen / n for n, f, seen in zip(ends, first, lens))
        else:
            pairs = keys * c["n_q"]
        values = 2 * c["batch"] * c["n_q"] * c["heads"] * 2 * c["dim"] + 2 * keys * c["kv_heads"] * 2 * c["dim"]
        more = 8 * c["batch"] * c["n_k"] if c["keys"] == "mask" else 0
        # two maps' scores, and the product of their difference with the values
        return {"bytes": values * e + more, "flops": 8.0 * c["dim"] * c["heads"] * pairs}
    if c["op"] == "rotary":
        values = c["batch"] * c["tokens"] * (c["q_heads"] + c["k_heads"])
        return {"bytes": 2 * values * c["dim"] * e + 8 * c["batch"] * c["tokens"] * c["axes"], "flops": 3.0 * values * c["rotary_dim"]}
    values = c["batch"] * c["rows"] * c["dim"]
    return {"bytes": values * 2 * (e + SIZE[c["resid"]]) + 4 * c["dim"] * 3 + (4 * c["batch"] * c["dim"] if c["gate"] else 0), "flops": 16.0 * values}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "diff_attention":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        batch, n_q, h, w = q.shape
        n_k, hk, d = k.shape[1], k.shape[2], w // 2
        lam = math.exp(float(torch.dot(s["lambda_qk"][0].double(), s["lambda_qk"][1].double())))
        lam += s["lambda_init"] - math.exp(float(torch.dot(s["lambda_qk"][2].double(), s["lambda_qk"][3].double())))
        out = torch.zeros(batch, n_q, h, w, dtype=torch.float64, device=q.device)
        for b in range(batch):
            n = n_k if s["kv_lens"] is None else int(s["kv_lens"][b])
            hidden = torch.zeros(n_q, n, dtype=torch.bool, device=q.device)
            if s["mask"] is not None:
                hidden |= (s["mask"][b, :n] == 0)[None]
            if s["causal"] != "no":
                hidden |= torch.arange(n, device=q.device)[None] > torch.arange(n_q, device=q.device)[:, None] + (n - n_q if s["causal"] == "end" else 0)
            blind = hidden.all(-1, keepdim=True)
            for i in range(h):
                kv = i // (h // hk)
                maps = []
                for m in range(2):
                    x = q[b, :, i, m * d:(m + 1) * d] @ k[b, :n, kv, m * d:(m + 1) * d].T.contiguous() * d ** -0.5
                    maps.append(torch.softmax(x.masked_fill(hidden & ~blind, -math.inf), -1).masked_fill(blind, 0.0))
                o = (maps[0] - lam * maps[1]) @ v[b, :n, kv]
                if s["norm"] is not None:
                    o = (1 - s["lambda_init"]) * s["norm"].double() * o / (o.square().mean(-1, keepdim=True) + EPS_ATTENTION).sqrt()
                out[b, :, i] = o
        return out
    if s["op"] == "rotary":
        f = s["freqs"].double().reshape(-1)
        per_axis = s["freqs"].shape[-1]
        pos = s["positions"].double().reshape(s["q"].shape[0], s["q"].shape[1], -1).repeat_interleave(per_axis, -1)
        turn = torch.polar(torch.ones_like(pos), pos * f)[:, :, None]
        outs = []
        for x in [s["q"], s["k"]]:
            if x is None:
                continue
            x, p = x.double(), f.numel()
            if s["layout"] == "half":
                z = torch.complex(x[..., :p].contiguous(), x[..., p:2 * p].contiguous()) * turn
                r = torch.cat([z.real, z.imag], -1)
            else:
                r = torch.view_as_real(torch.view_as_complex(x[..., :2 * p].reshape(*x.shape[:-1], p, 2).contiguous()) * turn).flatten(-2)
            outs.append(torch.cat([r, x[..., 2 * p:]], -1))
        return outs

    def norm(x, w, b):
        mu = x.mean(-1, keepdim=True) if s["kind"] == "layer" else 0.0
        return (x - mu) / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + EPS_NORM) * w.double() + (0.0 if b is None else b.double())

    t = s["y"].double()
    t = t if s["post"] is None else norm(t, *s["post"])
    factor = torch.ones(t.shape[-1], dtype=torch.float64, device=t.device) if s["scale"] is None else s["scale"].double()
    factor = factor if s["gate"] is None else factor * s["gate"].double()[:, None]
    r = s["residual"].double() + factor * t
    return [r, norm(r, *s["pre"])]
