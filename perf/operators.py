"""Latent attention over a paged cache and rotary positions: the cases that are timed.

Four operators of this library belong together in a serving step that keeps one
latent vector a token instead of keys and values per head:

* ``rope``     rotary positions on q and k: pairs (2i, 2i+1) or (i, i + R/2), the
               leading R elements of a head, frequencies scaled for long contexts;
* ``append``   root-mean-square norm of the latent, rotation of the shared key
               part, and both written through the block table into the cache;
* ``decode``   attention in the absorbed form: the query is already in the latent
               space, keys are [latent | rotary part], values are the latent;
* ``prefill``  attention of a chunk of new tokens in the expanded form: keys and
               values per head are the latent times the up-projection.

``run`` computes the plain form in 32 bits, or calls the library where ``own``
is true; ``exact`` computes the definition in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decode step of 64 sequences, 64 query and 8 key heads of 128 (a 70B GQA layer)
        dict(name="rope 64 tokens", op="rope", tokens=64, heads=64, kv_heads=8, head_dim=128, rotary=128, half=False,
             scaling="none", dtype="fp16"),
        # a prefill chunk of 8 x 2048 tokens, 32 + 32 heads (a 7B MHA layer), context extended four times
        dict(name="rope 16k tokens", op="rope", tokens=16384, heads=32, kv_heads=32, head_dim=128, rotary=128, half=True,
             scaling="by_parts", dtype="bf16"),
        # the new tokens of one decode step, written to the cache
        dict(name="append 32 tokens", op="append", batch=32, mean=1, sigma=0.0, prefix=1000, latent=512, rope=64, page=16,
             half=False, norm=True, shape=1, dtype="fp16"),
        # a ragged prefill batch of about 16k tokens, written to the cache
        dict(name="append 16k tokens", op="append", batch=8, mean=2048, sigma=0.5, prefix=77, latent=512, rope=64, page=64,
             half=True, norm=True, shape=2, dtype="bf16"),
        # one user, a short context, 8 heads of a head-sharded layer: latency counts
        dict(name="decode 1 x 200", op="decode", batch=1, tokens=1, heads=8, mean=200, sigma=0.0, latent=512, rope=64,
             page=16, shape=3, dtype="fp16"),
        # the decode step of 64 sequences of mixed lengths, 64 heads
        dict(name="decode 64 x 2k", op="decode", batch=64, tokens=1, heads=64, mean=2250, sigma=0.6, latent=512, rope=64,
             page=16, shape=4, dtype="fp16"),
        # drafted tokens: four query tokens a sequence are scored at once
        dict(name="decode 16 x 4k, 4 drafted", op="decode", batch=16, tokens=4, heads=32, mean=4000, sigma=0.4, latent=512,
             rope=64, page=16, shape=5, dtype="bf16"),
        # one very long context
        dict(name="decode 1 x 128k", op="decode", batch=1, tokens=1, heads=32, mean=131071, sigma=0.0, latent=512, rope=64,
             page=64, shape=6, dtype="bf16"),
        # long contexts under memory churn
        dict(name="decode 24 x 16k", op="decode", batch=24, tokens=1, heads=64, mean=16384, sigma=0.3, latent=512, rope=64,
             page=64, shape=7, dtype="fp16"),
        # short prompts behind a shared prefix
        dict(name="prefill 3 x 45", op="prefill", batch=3, mean=45, sigma=0.8, prefix=500, heads=32, latent=512, rope=64,
             page=16, shape=8, dtype="fp16"),
        # chunked prefill of 8 x 2048 tokens, 32 heads
        dict(name="prefill 8 x 2048", op="prefill", batch=8, mean=2048, sigma=0.0, prefix=0, heads=32, latent=512, rope=64,
             page=16, shape=9, dtype="fp16"),
        # a chunk late in long documents, a smaller latent, heads of one of several GPUs
        dict(name="prefill 2 x 1000 at 14k", op="prefill", batch=2, mean=1000, sigma=0.1, prefix=14000, heads=16, latent=256,
             rope=32, page=64, shape=10, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "append", "decode", "prefill"])
    dtype = rng.choice(["fp16", "bf16"])
    shape = rng.randrange(1 << 20)
    if op == "rope":
        head_dim = rng.choice([64, 96, 128, 192, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 5, 8])
        return dict(op=op, tokens=_log_int(rng, 1, min(16384, 16384 * 64 * 128 // ((heads + kv_heads) * head_dim))),
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary=rng.choice([r for r in (32, 64, head_dim // 2, head_dim) if r <= head_dim]),
                    half=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "by_parts", "by_wavelength"]), dtype=dtype)
    latent, rope = rng.choice([(512, 64), (512, 64), (256, 64), (256, 32), (384, 64), (128, 16)])
    page = rng.choice([16, 32, 64])
    sigma = rng.choice([0.0, 0.3, 0.8])
    if op == "append":
        batch = _log_int(rng, 1, 64)
        return dict(op=op, batch=batch, mean=_log_int(rng, 1, 10000 // batch), sigma=sigma, prefix=rng.choice([0, 5, 1000]),
                    latent=latent, rope=rope, page=page, half=rng.random() < 0.5, norm=rng.random() < 0.7, shape=shape,
                    dtype=dtype)
    if op == "decode":
        batch, tokens = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 7])
        heads = rng.choice([1, 8, 16, 20, 32, 64, 128]) if tokens == 1 else rng.choice([5, 8, 16, 32])
        return dict(op=op, batch=batch, tokens=tokens, heads=heads, mean=_log_int(rng, 1, min(100000, 180000 // batch)),
                    sigma=sigma, latent=latent, rope=rope, page=page, shape=shape, dtype=dtype)
    batch, heads = rng.choice([1, 2, 3, 5, 8]), rng.choice([4, 7, 8, 16, 32])
    return dict(op=op, batch=batch, mean=_log_int(rng, 1, 1800 // batch + 100), sigma=sigma,
                prefix=rng.choice([0, 3, _log_int(rng, 10, 16000 // batch)]), heads=heads, latent=latent, rope=rope, page=page,
                shape=shape, dtype=dtype)


# ------------------------------------------------------------------ sizes of a case


def _lengths(case, mean):
    """The batch's lengths: `mean` each, or lognormal around it, the same for every seed of the case."""
    r = random.Random(case["shape"])
    out = []
    for _ in range(case["batch"]):
        k = math.exp(r.gauss(0.0, case["sigma"]) - case["sigma"] ** 2 / 2) if case["sigma"] else 1.0
        out.append(max(1, min(int(mean * k), 4 * mean)))
    return out


def _sequences(case):
    """(tokens in the cache after the call, new tokens) of each sequence."""
    if case["op"] == "decode":
        lens = _lengths(case, case["mean"])
        return lens, [case["tokens"]] * case["batch"]
    new = _lengths(case, case["mean"])
    return [case["prefix"] + n for n in new], new


_SCALINGS = {  # for contexts four times as long as the 4096 positions of the base
    "none": dict(),
    "linear": dict(scaling="linear", factor=4.0),
    "by_parts": dict(scaling="by_parts", factor=4.0, original_len=4096, low=1.0, high=32.0),
    "by_wavelength": dict(scaling="by_wavelength", factor=8.0, original_len=8192, low=1.0, high=4.0),
}


def work(case):
    """Inputs read once, outputs written once; products and sums of the definition."""
    if case["op"] == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["head_dim"] * 2 + 4 * case["tokens"], "flops": 3 * n * case["rotary"]}
    lens, new = _sequences(case)
    width = case["latent"] + case["rope"]
    pages = sum(-(-n // case["page"]) for n in lens)
    if case["op"] == "append":
        return {"bytes": 2 * sum(new) * width * 2 + 4 * (sum(new) + 2 * case["batch"]),
                "flops": sum(new) * (4 * case["latent"] + 3 * case["rope"])}
    if case["op"] == "decode":
        rows = case["batch"] * case["tokens"] * case["heads"]
        pairs = sum(max(0, n - t) for n in lens for t in range(case["tokens"]))
        return {"bytes": 2 * sum(lens) * width + 2 * rows * (width + case["latent"]) + 4 * rows + 4 * pages,
                "flops": 2 * pairs * case["heads"] * (width + case["latent"])}
    rows = sum(new) * case["heads"]
    pairs = sum(n * (total - n) + n * (n + 1) // 2 for total, n in zip(lens, new))
    return {"bytes": 2 * sum(lens) * width + 2 * case["heads"] * 256 * case["latent"] + 2 * rows * (256 + case["rope"]) + 4 * pages,
            "flops": 2 * sum(lens) * case["heads"] * 256 * case["latent"] + 2 * pairs * case["heads"] * (256 + case["rope"])}


# ------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    state = dict(case=case, seed=seed)
    if case["op"] == "rope":
        state["q"] = normal(case["tokens"], case["heads"], case["head_dim"])
        state["k"] = normal(case["tokens"], case["kv_heads"], case["head_dim"])
        # positions of a batch in flight: anywhere in a context of 128k
        state["positions"] = torch.randint(0, 131072, (case["tokens"],), generator=g, device="cuda", dtype=torch.int32)
        if own:
            from vulcan_b200 import RotaryEmbedding
            state["rotary"] = RotaryEmbedding(case["rotary"], theta=10000.0, layout="half" if case["half"] else "interleaved",
                                              **_SCALINGS[case["scaling"]])
        return state

    # a pool of one layer whose pages the sequences own in random order
    lens, new = _sequences(case)
    latent, rope, page, batch = case["latent"], case["rope"], case["page"], case["batch"]
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu()
    tables = torch.full((batch, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = perm[at:at + n]
        at += n
    state["tables"] = tables.cuda()
    state["pages"] = normal(1, total, page, latent + rope)
    state["tokens"] = sum(new)
    state["longest_chunk"], state["longest"] = max(new), max(lens)
    state["positions"] = torch.tensor([n - k for n, k in zip(lens, new)], dtype=torch.int32).cuda()
    state["offsets"] = torch.tensor([0] + [sum(new[:b + 1]) for b in range(batch)], dtype=torch.int32).cuda()
    state["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
    # for the plain form: which sequence and position each new token has
    state["token_seq"] = torch.repeat_interleave(torch.arange(batch), torch.tensor(new)).cuda()
    state["token_pos"] = torch.cat([torch.arange(n - k, n) for n, k in zip(lens, new)]).cuda()
    if case["op"] == "append":
        # rows of the down-projection: latent and shared key part side by side
        state["kv"] = normal(sum(new), latent + rope)
        state["weight"] = (1.0 + 0.1 * torch.randn(latent, generator=g, device="cuda")).to(dtype)
    elif case["op"] == "decode":
        state["q_latent"] = normal(batch, case["tokens"], case["heads"], latent, std=0.5)
        state["q_rope"] = normal(batch, case["tokens"], case["heads"], rope)
    else:
        state["q"] = normal(sum(new), case["heads"], 128 + rope)
        state["w_kv"] = normal(case["heads"] * 256, latent, std=latent ** -0.5)
    if own:
        from vulcan_b200 import LatentKVPool, RotaryEmbedding
        state["pool"] = LatentKVPool(1, latent, rope, total, page_tokens=page, dtype=dtype, storage=state["pages"])
        state["rotary"] = RotaryEmbedding(rope, theta=10000.0, layout="half" if case.get("half") else "interleaved")
    return state


# ------------------------------------------------------------------ plain forms, 32 bits


def _frequencies(rotary, scaling):
    """Angle per position of each pair, in 64 bits: angles of far positions lose what matters in 32."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
    f = 10000.0 ** (-2.0 * i / rotary)
    s = _SCALINGS[scaling]
    if scaling == "linear":
        f = f / s["factor"]
    elif scaling == "by_parts":
        turns = [rotary * math.log(s["original_len"] / (2 * math.pi * n)) / (2 * math.log(10000.0)) for n in (s["high"], s["low"])]
        first, last = max(math.floor(turns[0]), 0), min(math.ceil(turns[1]), rotary // 2 - 1)
        ramp = ((i - first) / max(last - first, 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / s["factor"] * ramp
    elif scaling == "by_wavelength":
        blend = ((s["original_len"] * f / (2 * math.pi) - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        f = (1 - blend) * f / s["factor"] + blend * f
    return f, (0.1 * math.log(s["factor"]) + 1.0) if scaling == "by_parts" else 1.0


def _rotate(x, positions, rotary, half, scaling):
    """x: [tokens, heads, D] in 32 bits; the leading `rotary` elements of each head turn."""
    f, magnitude = _frequencies(rotary, scaling)
    angle = positions.double()[:, None] * f
    cos, sin = (angle.cos() * magnitude).float()[:, None], (angle.sin() * magnitude).float()[:, None]
    part = x[..., :rotary]
    if half:
        a, b = part[..., :rotary // 2], part[..., rotary // 2:]
        part = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([part, x[..., rotary:]], -1)


def _plain_append(s):
    case, latent = s["case"], s["case"]["latent"]
    c = s["kv"][:, :latent].float()
    if case["norm"]:
        c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    k = _rotate(s["kv"][:, None, latent:].float(), s["token_pos"], case["rope"], case["half"], "none")[:, 0]
    page = s["tables"][s["token_seq"], s["token_pos"] // case["page"]].long()
    s["pages"][0, page, s["token_pos"] % case["page"]] = torch.cat([c, k], -1).to(s["pages"].dtype)
    return s["pages"]


def _gathered(s):
    """The cached rows of every sequence, [batch, longest, latent + rope] in 32 bits, zeros behind the ends."""
    rows = s["pages"][0][s["tables"].clamp(min=0).long()].flatten(1, 2)[:, :s["longest"]].float()
    inside = torch.arange(rows.shape[1], device="cuda")[None, :] < s["lens"][:, None]
    return torch.where(inside[..., None], rows, 0.0)


def _softmax(scores, visible):
    """Weights and log of the sum; a row without a visible key has weights of zero."""
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0), (top + torch.log(total))[..., 0]


def _plain_decode(s):
    case = s["case"]
    rows, t = _gathered(s), case["tokens"]
    q = torch.cat([s["q_latent"], s["q_rope"]], -1).float()
    scores = torch.matmul(q.flatten(1, 2), rows.transpose(1, 2)).view(*q.shape[:3], -1) * (128 + case["rope"]) ** -0.5
    limit = s["lens"][:, None] - (t - 1 - torch.arange(t, device="cuda"))  # keys that query token t sees
    visible = torch.arange(rows.shape[1], device="cuda") < limit[:, :, None, None]
    p, lse = _softmax(scores, visible)
    out = torch.matmul(p.flatten(1, 2), rows[..., :case["latent"]]).view(*q.shape[:3], -1)
    return out.to(s["pages"].dtype), lse


def _plain_prefill(s):
    case, latent, heads = s["case"], s["case"]["latent"], s["case"]["heads"]
    rows, w = _gathered(s), s["w_kv"].float()
    kv = torch.matmul(rows[..., :latent], w.t()).unflatten(-1, (heads, 256)).permute(0, 2, 1, 3)  # [batch, heads, longest, 256]
    keys = torch.cat([kv[..., :128], rows[:, None, :, latent:].expand(-1, heads, -1, -1)], -1)
    # the ragged chunk, padded: slot (sequence, index in the chunk) of each token
    index = s["token_pos"] - s["positions"][s["token_seq"]]
    q = torch.zeros(case["batch"], s["longest_chunk"], heads, 128 + case["rope"], device="cuda")
    q[s["token_seq"], index] = s["q"].float()
    scores = torch.matmul(q.transpose(1, 2), keys.transpose(2, 3)) * (128 + case["rope"]) ** -0.5
    row_pos = s["positions"][:, None] + torch.arange(q.shape[1], device="cuda")
    visible = torch.arange(rows.shape[1], device="cuda") <= row_pos[:, None, :, None]
    out = torch.matmul(_softmax(scores, visible)[0], kv[..., 128:])
    return out.transpose(1, 2)[s["token_seq"], index].to(s["pages"].dtype)


def run(s):
    case = s["case"]
    if case["op"] == "rope":
        if own:
            return s["rotary"].apply(s["q"], s["positions"], k=s["k"])
        return tuple(_rotate(x.float(), s["positions"], case["rotary"], case["half"], case["scaling"]).to(x.dtype)
                     for x in (s["q"], s["k"]))
    if case["op"] == "append":
        if not own:
            return _plain_append(s)
        s["pool"].append(0, s["kv"][:, :case["latent"]], s["kv"][:, case["latent"]:], s["tables"], s["positions"],
                         offsets=s["offsets"], norm_weight=s["weight"] if case["norm"] else None, eps=1e-6, rope=s["rotary"])
        return s["pages"]
    if case["op"] == "decode":
        if not own:
            return _plain_decode(s)
        return s["pool"].decode(0, s["q_latent"], s["q_rope"], s["tables"], s["lens"], scale=(128 + case["rope"]) ** -0.5,
                                return_lse=True)
    if not own:
        return _plain_prefill(s)
    return s["pool"].prefill(0, s["q"], s["w_kv"], s["tables"], s["positions"], offsets=s["offsets"],
                             max_tokens=s["longest_chunk"], max_seq_len=s["longest"])


# ------------------------------------------------------------------ the definitions, 64 bits


def _turn(x, positions, rotary, half, scaling):
    """Rotation as a product of complex numbers, pair by pair."""
    s, magnitude, speed = _SCALINGS[scaling], 1.0, []
    for i in range(rotary // 2):
        w = math.exp(-math.log(10000.0) * 2 * i / rotary)
        if scaling == "linear":
            w /= s["factor"]
        elif scaling == "by_parts":
            def pair_of(turns):  # the pair that makes this many turns within the original context
                return rotary * math.log(s["original_len"] / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
            lo, hi = max(math.floor(pair_of(s["high"])), 0), min(math.ceil(pair_of(s["low"])), rotary // 2 - 1)
            share = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = share * w / s["factor"] + (1.0 - share) * w
            magnitude = 1.0 + math.log(s["factor"]) / 10
        elif scaling == "by_wavelength":
            length = 2 * math.pi / w
            if length > s["original_len"] / s["low"]:
                w /= s["factor"]
            elif length >= s["original_len"] / s["high"]:
                share = (s["original_len"] / length - s["low"]) / (s["high"] - s["low"])
                w = (1 - share) * w / s["factor"] + share * w
        speed.append(w)
    angle = positions.double()[:, None, None] * torch.tensor(speed, dtype=torch.float64, device="cuda")
    unit = torch.polar(torch.full_like(angle, magnitude), angle)
    y = x.double().clone()
    re, im = (slice(0, rotary // 2), slice(rotary // 2, rotary)) if half else (slice(0, rotary, 2), slice(1, rotary, 2))
    z = torch.complex(y[..., re].contiguous(), y[..., im].contiguous()) * unit
    y[..., re], y[..., im] = z.real, z.imag
    return y


def _cached(s, b, n):
    """Rows 0..n-1 of sequence b in 64 bits."""
    ids = s["tables"][b, :-(-n // s["case"]["page"])].long()
    return s["pages"][0, ids].reshape(-1, s["pages"].shape[-1])[:n].double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return tuple(_turn(x, s["positions"], case["rotary"], case["half"], case["scaling"]) for x in (s["q"], s["k"]))
    latent = case["latent"]
    lens, new = _sequences(case)
    if case["op"] == "append":
        want = s["pages"].double()
        c, k = s["kv"].double().split([latent, case["rope"]], -1)
        if case["norm"]:
            c = c / torch.sqrt(c.square().sum(-1, keepdim=True) / latent + 1e-6) * s["weight"].double()
        k = _turn(k[:, None], s["token_pos"], case["rope"], case["half"], "none")[:, 0]
        at = 0
        for b, n in enumerate(new):
            pos = torch.arange(lens[b] - n, lens[b], device="cuda")
            ids = s["tables"][b].long()[pos // case["page"]]
            want[0, ids, pos % case["page"], :latent] = c[at:at + n]
            want[0, ids, pos % case["page"], latent:] = k[at:at + n]
            at += n
        return want
    scale = 1.0 / math.sqrt(128 + case["rope"])
    if case["op"] == "decode":
        shape = (case["batch"], case["tokens"], case["heads"])
        out = torch.zeros(*shape, latent, dtype=torch.float64, device="cuda")
        lse = torch.full(shape, -math.inf, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            rows = _cached(s, b, n)
            for t in range(case["tokens"]):
                seen = rows[:max(0, n - (case["tokens"] - 1 - t))]
                if len(seen):
                    q = torch.cat([s["q_latent"][b, t], s["q_rope"][b, t]], -1).double()
                    a = scale * torch.einsum("hd,kd->hk", q, seen)
                    lse[b, t] = torch.logsumexp(a, -1)
                    out[b, t] = torch.einsum("hk,kd->hd", torch.exp(a - lse[b, t][:, None]), seen[:, :latent])
        return out, lse
    out = torch.zeros(s["tokens"], case["heads"], 128, dtype=torch.float64, device="cuda")
    at = 0
    for b, n in enumerate(new):
        rows, first = _cached(s, b, lens[b]), lens[b] - n
        hidden = torch.arange(lens[b], device="cuda")[None] > torch.arange(first, lens[b], device="cuda")[:, None]
        for h in range(case["heads"]):
            up = s["w_kv"][h * 256:(h + 1) * 256].double()
            q = s["q"][at:at + n, h].double()
            a = torch.einsum("td,kd->tk", q[:, :128], torch.einsum("kc,dc->kd", rows[:, :latent], up[:128]))
            a = scale * (a + torch.einsum("td,kd->tk", q[:, 128:], rows[:, latent:]))
            a = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
            out[at:at + n, h] = torch.einsum("tk,kd->td", a, torch.einsum("kc,dc->kd", rows[:, :latent], up[128:]))
        at += n
    return out
