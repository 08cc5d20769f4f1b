"""Measured cases of the target stack in few bits: attention over a 4-bit cache,
the commit into it, and projections in 8-bit floating point.

  attn    packed tree attention of one layer over prefixes held in 4 bits
          (e2m1 elements, one power-of-two scale for 32 of them), the wave's own
          rows in bf16
  commit  every layer's kept rows into the 4-bit arena, then the arena's values
          (a pool's `keys` / `values` views)
  proj    a projection in e4m3: the activations get a scale for each row and 128
          columns from their producer (residual add and RMSNorm, SiLU * up, or
          the rows as they are), the weight has one for each 128 x 128 block

`own` false: the plain forms, in elementary torch operations and fp32.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BF16 = torch.bfloat16
F8 = torch.float8_e4m3fn
DEVICE = "cuda:0"
EPS = 1e-6
TINY = 2.0 ** -100  # the least maximum that a row block's scale is made from


def listed():
    return [
        # Smallest wave: four 16-node trees of a test-size model.
        {"name": "attn4_tiny", "kind": "attn", "requests": 4, "lo": 32, "hi": 96, "tiers": "16",
         "budget": 64, "hq": 4, "hkv": 2, "dim": 64, "tree": "random", "wave": 1},
        # Plain decoding: one row a request.
        {"name": "attn4_step", "kind": "attn", "requests": 48, "lo": 500, "hi": 4000,
         "tiers": "1", "budget": 48, "hq": 32, "hkv": 8, "dim": 128, "tree": "random",
         "wave": 2},
        # The ordinary verification wave: 64 requests, 2048-row budget.
        {"name": "attn4_64req", "kind": "attn", "requests": 64, "lo": 512, "hi": 4096,
         "tiers": "16,32,64,128", "budget": 2048, "hq": 32, "hkv": 8, "dim": 128,
         "tree": "random", "wave": 3},
        # Long contexts, what the four bits are for.
        {"name": "attn4_long", "kind": "attn", "requests": 32, "lo": 8192, "hi": 32768,
         "tiers": "1,16,32,64", "budget": 1024, "hq": 32, "hkv": 8, "dim": 128,
         "tree": "random", "wave": 4},
        # The accepted rows of a wave into the arena of 36 layers.
        {"name": "commit4_wave", "kind": "commit", "requests": 64, "layers": 36, "hkv": 8,
         "dim": 128, "rows": 32, "keep": 9, "capacity": 16, "wave": 5},
        # Prefilled prompts moved into the arena: every row of each is kept.
        {"name": "commit4_prompts", "kind": "commit", "requests": 8, "layers": 4, "hkv": 8,
         "dim": 128, "rows": 1500, "keep": 0, "capacity": 1600, "wave": 6},
        # One token's attention output through the output projection.
        {"name": "proj8_one_row", "kind": "proj", "of": "rows", "rows": 1, "k": 4096, "n": 4096},
        # A small wave into the q/k/v projection.
        {"name": "proj8_qkv_64", "kind": "proj", "of": "norm", "rows": 64, "k": 2560, "n": 6144},
        # Ragged sizes: no multiple of a tile or of 128 anywhere.
        {"name": "proj8_odd", "kind": "proj", "of": "rows", "rows": 333, "k": 2568, "n": 50257},
        # A lightly loaded server's wave out of the feed-forward block.
        {"name": "proj8_down_512", "kind": "proj", "of": "silu", "rows": 512, "k": 12288,
         "n": 4096},
        # A full wave out of it, and into it: the largest product.
        {"name": "proj8_down_2048", "kind": "proj", "of": "silu", "rows": 2048, "k": 12288,
         "n": 4096},
        {"name": "proj8_gateup_2048", "kind": "proj", "of": "norm", "rows": 2048, "k": 4096,
         "n": 24576},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above, odd sizes among them."""
    kind = rng.choices(["attn", "commit", "proj"], [5, 2, 6])[0]
    if kind == "attn":
        tree = rng.choice(["random", "random", "chain"])
        tiers = rng.choice(["1,16,32,64", "16,32,64,128", "1", "7,33,65"] if tree == "random"
                           else ["1,7,64,200", "256"])
        most = int(tiers.split(",")[-1])
        hq, hkv = rng.choice([(32, 8), (32, 8), (4, 2), (16, 8), (64, 8), (16, 16), (32, 2)])
        requests = _log_int(rng, 1, 64)
        hi = _log_int(rng, 40, min(32768, 600000 // requests,
                                   2000000000 // (requests * most * hq)))
        return {"kind": kind, "requests": requests, "lo": max(1, hi // rng.choice([1, 2, 4, 40])),
                "hi": hi, "tiers": tiers, "budget": most * requests, "hq": hq, "hkv": hkv,
                "dim": rng.choice([64, 128, 128]), "tree": tree, "wave": rng.randrange(1 << 30)}
    if kind == "commit":
        prompts = rng.random() < 0.4
        rows = _log_int(rng, 10, 3000) if prompts else rng.choice([9, 16, 32])
        keep = 0 if prompts else rng.choice([1, 2, 9])
        hkv, dim = rng.choice([(2, 64), (8, 128), (8, 128), (3, 64), (16, 128)])
        layers = rng.choice([1, 2, 4]) if prompts else rng.choice([1, 2, 36])
        capacity = (rows if prompts else keep) + rng.choice([1, 7, 20])
        return {"kind": kind, "requests": _log_int(rng, 1, min(
                    64, 76000000 // (capacity * layers * hkv * dim * 2))),
                "layers": layers, "hkv": hkv, "dim": dim, "rows": rows, "keep": keep,
                "capacity": capacity, "wave": rng.randrange(1 << 30)}
    of = rng.choice(["rows", "norm", "silu"])
    k = rng.choice([256, 768, 2560, 4096, 4096, 12288 if of != "norm" else 8192,
                    8 * _log_int(rng, 12, 1000)])
    rows = _log_int(rng, 1, 4096)
    most = max(64, min(50257, int(2.05e11 / (k * rows))))
    n = rng.choice([v for v in (768, 4096, 6144, 24576) if v <= most] or [64])
    return {"kind": kind, "of": of, "rows": rows, "k": k,
            "n": n if rng.random() < 0.6 else _log_int(rng, 64, most)}


# --------------------------------------------------------------------------
# shapes of a case (from its values alone)
# --------------------------------------------------------------------------

def _tree(kind, nodes, rng):
    """Parents of a tree: a chain, or breadth first with 1 to 4 children a node."""
    if kind == "chain":
        return list(range(-1, nodes - 1))
    parents, at = [-1], 0
    while len(parents) < nodes:
        parents += [at] * min(int(rng.integers(1, 5)), nodes - len(parents))
        at += 1
    return parents


def _wave(c):
    """Row offsets, prefix starts and lengths, parents and capacity of a wave."""
    rng = np.random.default_rng(c["wave"])
    n, tiers = c["requests"], [int(t) for t in c["tiers"].split(",")]
    lengths = np.floor(np.exp(rng.uniform(math.log(c["lo"]), math.log(c["hi"] + 1), n)))
    lengths = np.minimum(lengths, c["hi"]).astype(np.int32)
    size = rng.choice(tiers, size=n)
    while size.sum() > c["budget"]:
        big = int(size.argmax())
        size[big] = tiers[tiers.index(int(size[big])) - 1]
    parents = [_tree(c["tree"], int(s), rng) for s in size]
    offset = np.concatenate([[0], np.cumsum(size)]).astype(np.int32)
    capacity = (int(lengths.max()) + 9 + 63) // 64 * 64
    return offset, np.arange(n, dtype=np.int64) * capacity, lengths, parents, capacity


def _visible(parents):
    """[T, T] of one tree: which nodes are a node's ancestors or itself."""
    seen = np.eye(len(parents), dtype=bool)
    for k in range(1, len(parents)):
        seen[k] |= seen[parents[k]]
    return seen


def _keeps(c):
    """Kept rows of each request (ascending, the root among them), and the
    lengths they are appended to."""
    rng = np.random.default_rng(c["wave"])
    if not c["keep"]:
        sizes = rng.integers(max(1, c["rows"] // 2), c["rows"] + 1, c["requests"])
        return sizes, None, np.zeros(c["requests"], np.int32)
    lens = rng.integers(1, min(c["keep"], c["rows"]) + 1, c["requests"])
    rows = np.full((c["requests"], c["keep"]), -1, np.int32)
    for i, k in enumerate(lens):
        rows[i, :k] = np.sort(np.concatenate([[0], 1 + rng.permutation(c["rows"] - 1)[:k - 1]]))
    return lens, rows, rng.integers(0, c["capacity"] - c["keep"] + 1, c["requests"]).astype(np.int32)


def work(c):
    if c["kind"] == "attn":
        offset, _, lengths, parents, _ = _wave(c)
        rows = np.diff(offset)
        pairs = int((rows * lengths).sum()) + sum(int(_visible(p).sum()) for p in parents)
        d = c["dim"]
        cache = int(lengths.sum()) * 2 * c["hkv"] * (d // 2 + d // 32)
        return {"bytes": cache + 2 * int(offset[-1]) * d * (2 * c["hq"] + 2 * c["hkv"]),
                "flops": 4 * c["hq"] * d * pairs}
    if c["kind"] == "commit":
        token = 2 * c["layers"] * c["hkv"] * c["dim"]
        packed = token // 2 + token // 32
        kept, whole = int(_keeps(c)[0].sum()), c["requests"] * c["capacity"]
        return {"bytes": kept * (2 * token + packed) + whole * (2 * token + packed), "flops": 0}
    rows, k, n = c["rows"], c["k"], c["n"]
    read = {"rows": 2, "norm": 6, "silu": 4}[c["of"]]
    return {"bytes": n * k + rows * (read * k + 2 * n), "flops": 2 * rows * n * k}


# --------------------------------------------------------------------------
# states
# --------------------------------------------------------------------------

def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)


def _mx4_pack(x):
    """Codes [..., D/2] and scales [..., D/32] of bf16 rows.  A block's scale is the
    least power of two of which its largest element is at most 7 times; codes 1 to
    252 stand for 2^(code - 127).  Elements go to the nearest of 0, 1/2, 1, 3/2, 2,
    3, 4, 6 times the scale, ties to the even code.  A block with an infinity or a
    NaN has scale 255 (NaN) and codes 0."""
    y = x.float().unflatten(-1, (-1, 32))
    bits = y.abs().amax(-1, keepdim=True).view(torch.int32)
    bad = bits >= 0x7F800000
    e = (((bits + 0x1FFFFF) >> 23) - 2).clamp(1, 252)
    z = y.abs() * ((254 - e) << 23).view(torch.float32)
    t = (z > 0.25).to(torch.uint8)
    t += z >= 0.75
    t += z > 1.25
    t += z >= 1.75
    t += z > 2.5
    t += z >= 3.5
    t += z > 5
    t += (y < 0) * torch.tensor(8, dtype=torch.uint8, device=x.device)
    t = torch.where(bad, torch.zeros_like(t), t).flatten(-2)
    scales = torch.where(bad, 255, e).squeeze(-1).to(torch.uint8)
    return t[..., 0::2] | (t[..., 1::2] << 4), scales


def _mx4_values(codes, scales):
    """fp32 values of codes and scales."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    t = (c & 7).float()
    v = 0.5 * (t + (t - 4).relu()) + (t - 6).relu()
    v = torch.where(c > 7, -v, v).unflatten(-1, (-1, 32))
    s = (scales.to(torch.int32) << 23).view(torch.float32)
    s = torch.where(scales == 255, torch.nan, s)
    return (v * s.unsqueeze(-1)).flatten(-2)


def _prepare_attn(c, g):
    offset, start, lengths, parents, capacity = _wave(c)
    n, rows, d = c["requests"], int(offset[-1]), c["dim"]
    tokens = n * capacity
    within = (torch.arange(capacity, device=DEVICE)[None] < _dev(lengths)[:, None]).view(-1)
    s = {"dim": d, "group": c["hq"] // c["hkv"],
         "q": 1.5 * torch.randn((rows, c["hq"], d), generator=g, device=DEVICE, dtype=BF16)}
    for name in ("k", "v"):
        x = torch.randn((c["hkv"], tokens, d), generator=g, device=DEVICE, dtype=BF16)
        codes, scales = _mx4_pack(x)
        scales[:, ~within] = 255  # what lies behind a request's last token is no value
        s[name + "_codes"], s[name + "_scales"] = codes, scales
        s[name + "_tree"] = torch.randn((rows, c["hkv"], d), generator=g, device=DEVICE,
                                        dtype=BF16)
    most, deep = int(np.diff(offset).max()), int(lengths.max())
    # A padded wave: request i's row t, its keys (prefix, then tree), what sees what.
    at = offset[:-1, None] + np.minimum(np.arange(most)[None], np.diff(offset)[:, None] - 1)
    seen = np.zeros((n, most, most), bool)
    for i, p in enumerate(parents):
        seen[i, :len(p), :len(p)] = _visible(p)
    seen |= np.eye(most, dtype=bool)
    live = torch.arange(deep, device=DEVICE)[None] < _dev(lengths)[:, None]
    s["live"] = live
    s["rows_of"] = _dev(at.astype(np.int64))
    s["keys_of"] = torch.where(live, torch.arange(deep, device=DEVICE)[None]
                               + _dev(start)[:, None], 0)
    s["seen"] = torch.cat([live[:, None].expand(n, most, deep), _dev(seen)], 2)
    owner = np.repeat(np.arange(n), np.diff(offset))
    s["back"] = _dev((owner * most + np.arange(rows) - offset[owner]).astype(np.int64))
    s["meta"] = (_dev(offset), _dev(start), _dev(lengths),
                 _dev(np.concatenate(parents).astype(np.int32)))
    if own:
        from specgrove_amd import ops
        s["plan"] = ops.plan_attention_mx4(offset, lengths, c["hq"], c["hkv"], d).to(DEVICE)
    return s


def _prepare_commit(c, g):
    lens, keep, lengths = _keeps(c)
    n, cap = c["requests"], c["capacity"]
    sizes = lens if keep is None else np.full(n, c["rows"])
    offset = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    shape = (2, c["layers"], c["hkv"])
    tree = torch.randn((*shape, int(offset[-1]), c["dim"]), generator=g, device=DEVICE,
                       dtype=BF16)
    old = torch.randn((*shape, n * cap, c["dim"]), generator=g, device=DEVICE, dtype=BF16)
    codes, scales = _mx4_pack(old)
    start = np.arange(n, dtype=np.int64) * cap
    owner = np.repeat(np.arange(n), lens)
    nth = np.arange(int(lens.sum())) - np.repeat(np.cumsum(lens) - lens, lens)
    local = nth if keep is None else keep[owner, nth]
    s = {"tree": tree, "codes": codes, "scales": scales, "capacity": cap,
         "from": _dev((offset[owner] + local).astype(np.int64)),
         "to": _dev(start[owner] + lengths[owner] + nth),
         "offset": _dev(offset), "start": _dev(start), "lengths": _dev(lengths),
         "keep": None if keep is None else _dev(keep), "keep_len": _dev(lens.astype(np.int32))}
    if own:
        from specgrove_amd import ops
        parts = [(t, i) for i in (0, 1) for t in (codes, scales)] + [(tree, 0), (tree, 1)]
        s["pointers"] = [ops.pointer_array(list(t[i].unbind(0)), DEVICE) for t, i in parts]
    return s


def _prepare_proj(c, g):
    rows, k, n = c["rows"], c["k"], c["n"]
    w = torch.randn((n, k), generator=g, device=DEVICE) / math.sqrt(k)
    pad = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128))
    blocks = pad.unflatten(0, (-1, 128)).unflatten(-1, (-1, 128))
    ws = blocks.abs().amax((1, 3)) / 448
    wq = (blocks / ws[:, None, :, None]).flatten(2).flatten(0, 1)[:n, :k].to(F8).contiguous()
    s = {"of": c["of"], "weight": wq, "weight_scales": ws}
    if c["of"] == "silu":
        s["x"] = 2 * torch.randn((rows, 2 * k), generator=g, device=DEVICE, dtype=BF16)
    else:
        # A few columns larger than the others, as hidden states have them.
        x = torch.randn((rows, k), generator=g, device=DEVICE)
        s["x"] = (x * (1 + 20 * (torch.rand(k, generator=g, device=DEVICE) < 0.01))).to(BF16)
    if c["of"] == "norm":
        s["residual"] = 3 * torch.randn((rows, k), generator=g, device=DEVICE, dtype=BF16)
        s["norm"] = 1 + 0.1 * torch.randn(k, generator=g, device=DEVICE, dtype=BF16)
    if own:
        from specgrove_amd import ops
        s["packed"] = ops.pack_fp8_weight(wq, ws)
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"kind": case["kind"],
            **{"attn": _prepare_attn, "commit": _prepare_commit,
               "proj": _prepare_proj}[case["kind"]](case, g)}


# --------------------------------------------------------------------------
# passes
# --------------------------------------------------------------------------

def _plain_attn(s):
    d, group = s["dim"], s["group"]

    def keys(name):
        codes = s[name + "_codes"][:, s["keys_of"]]
        x = _mx4_values(codes, s[name + "_scales"][:, s["keys_of"]])
        x = torch.where(s["live"][:, :, None], x, 0)
        return torch.cat([x, s[name + "_tree"][s["rows_of"]].float().movedim(2, 0)], 2)

    q = s["q"][s["rows_of"]].float()                       # [n, T, Hq, D]
    n, most = q.shape[:2]
    q = q.unflatten(2, (-1, group)).permute(2, 0, 3, 1, 4).flatten(2, 3)  # [Hkv, n, G T, D]
    x = torch.matmul(q, keys("k").transpose(2, 3).contiguous())
    x = x.unflatten(2, (group, most)) * d ** -0.5
    x = x.masked_fill(~s["seen"][None, :, None], -torch.inf)
    x -= x.amax(-1, keepdim=True)
    x = x.exp_()
    x /= x.sum(-1, keepdim=True)
    out = torch.matmul(x.flatten(2, 3), keys("v")).unflatten(2, (group, most))
    out = out.permute(1, 3, 0, 2, 4).reshape(n * most, -1, d)
    return out[s["back"]].to(BF16)


def _run_attn(s):
    if own:
        from specgrove_amd import ops
        return ops.tree_attention_mx4(s["q"], s["k_codes"], s["k_scales"], s["v_codes"],
                                      s["v_scales"], s["k_tree"], s["v_tree"], *s["meta"],
                                      s["plan"])
    return _plain_attn(s)


def _run_commit(s):
    codes, scales, tree = s["codes"], s["scales"], s["tree"]
    if own:
        from specgrove_amd import ops
        lengths = s["lengths"].clone()
        ops.kv_commit_mx4(
            *s["pointers"], num_kv_heads=tree.shape[2], head_dim=tree.shape[4],
            code_head_stride=codes.stride(2), code_token_stride=codes.stride(3),
            scale_head_stride=scales.stride(2), scale_token_stride=scales.stride(3),
            tree_row_stride=tree.stride(3), tree_head_stride=tree.stride(2),
            row_offset=s["offset"], keep_rows=s["keep"], keep_len=s["keep_len"],
            prefix_start=s["start"], lengths=lengths, capacity=s["capacity"])
        return ops.kv_load_mx4(codes, scales), lengths
    new, by = _mx4_pack(tree[:, :, :, s["from"]])
    codes[:, :, :, s["to"]] = new
    scales[:, :, :, s["to"]] = by
    return _mx4_values(codes, scales).to(BF16), s["lengths"] + s["keep_len"]


def _plain_quantized(x):
    """Values of fp32 rows held in e4m3 with a scale for each row and 128 columns."""
    k = x.shape[1]
    b = torch.nn.functional.pad(x, (0, -k % 128)).unflatten(1, (-1, 128))
    most = b.abs().amax(2, keepdim=True).clamp_min(TINY)
    return ((b * (448 / most)).to(F8).float() * (most / 448)).flatten(1)[:, :k]


def _plain_weight(s):
    w, ws = s["weight"].float(), s["weight_scales"]
    n, k = w.shape
    return w * ws.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _run_proj(s):
    of, x = s["of"], s["x"]
    if own:
        from specgrove_amd import ops, target
        if of == "norm":
            rows, total = target.add_rmsnorm_fp8(x, s["norm"], EPS, s["residual"], want_sum=True)
            return ops.fp8_matmul(rows, s["packed"]), total
        rows = target.silu_mul_fp8(x) if of == "silu" else ops.quantize_fp8(x)
        return ops.fp8_matmul(rows, s["packed"])
    total = None
    if of == "norm":
        total = (x.float() + s["residual"].float()).to(BF16)  # the residual stream is bf16
        f = total.float()
        y = f * (1 / (f.square().mean(1, keepdim=True) + EPS).sqrt()) * s["norm"].float()
    elif of == "silu":
        gate, up = x.float().chunk(2, 1)
        y = gate / (1 + (-gate).exp()) * up
    else:
        y = x.float()
    out = torch.matmul(_plain_quantized(y), _plain_weight(s).T).to(BF16)
    return out if total is None else (out, total)


def run(state):
    return {"attn": _run_attn, "commit": _run_commit, "proj": _run_proj}[state["kind"]](state)


# --------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------

def _exact_values(codes, scales):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEVICE)
    table = torch.cat([table, -table])
    x = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.float64, device=DEVICE)
    x[..., 0::2] = table[(codes % 16).int()]
    x[..., 1::2] = table[(codes // 16).int()]
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=DEVICE), scales.double() - 127)
    return x * s.repeat_interleave(32, -1)


def _exact_attn(c, s):
    offset, start, lengths, parents, _ = _wave(c)
    out = []
    for i, p in enumerate(parents):
        a, b = int(offset[i]), int(offset[i + 1])
        span = slice(int(start[i]), int(start[i]) + int(lengths[i]))
        k, v = (torch.cat([_exact_values(s[x + "_codes"][:, span], s[x + "_scales"][:, span]),
                           s[x + "_tree"][a:b].double().transpose(0, 1)], 1) for x in "kv")
        q = s["q"][a:b].double().transpose(0, 1).reshape(c["hkv"], -1, c["dim"])
        score = (q @ k.transpose(1, 2).contiguous()) / math.sqrt(c["dim"])
        hidden = ~_dev(_visible(p)).repeat(c["hq"] // c["hkv"], 1)
        score[:, :, int(lengths[i]):].masked_fill_(hidden[None], -torch.inf)
        o = torch.softmax(score, 2) @ v
        out.append(o.reshape(c["hq"], b - a, c["dim"]).transpose(0, 1))
    return torch.cat(out)


def _exact_commit(c, s):
    values = _exact_values(s["codes"], s["scales"])
    x = s["tree"][:, :, :, s["from"]].double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    unit = torch.pow(2.0, torch.ceil(torch.log2((top / 7).clamp_min(2.0 ** -126))))
    y = (x / unit).abs()
    y = torch.where(y < 2, (2 * y).round() / 2, torch.where(y < 4, y.round(), 2 * (y / 2).round()))
    values[:, :, :, s["to"]] = (y.clamp_max(6) * x.sign() * unit).flatten(-2)
    return values, None


def _exact_proj(c, s):
    x, total = s["x"].double(), None
    if c["of"] == "norm":
        total = x + s["residual"].double()
        x = total.to(BF16).double()
        x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["norm"].double()
    elif c["of"] == "silu":
        x = torch.sigmoid(x[:, :c["k"]]) * x[:, :c["k"]] * x[:, c["k"]:]
    out = torch.zeros((c["rows"], c["n"]), dtype=torch.float64, device=DEVICE)
    for j in range(0, c["k"], 128):
        part = x[:, j:j + 128]
        unit = part.abs().amax(1, keepdim=True).clamp_min(TINY) / 448
        part = (part / unit).float().to(F8).double() * unit
        w = s["weight"][:, j:j + 128].double()
        w *= s["weight_scales"][:, j // 128].double().repeat_interleave(128)[:c["n"], None]
        out += part @ w.T
    return out if total is None else (out, total)


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "commit": _exact_commit, "proj": _exact_proj}[case["kind"]](case, s)
