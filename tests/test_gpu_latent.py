"""GPU tests of the latent cache: append, absorbed decode, expanded prefill, page
operations, and a run of them together, against the definitions in 64 bits.

Tolerances, from the roundings of each path (e = eps / 2 of the cache's type):

append   one rounding of a value whose fp32 arithmetic is within 2^-19 (21
         additions of squares, rsqrt, two products; the rotation as in
         test_gpu_rotary.py): (e + 2^-19) |want| + (|a| + |b|) 2^-19 + 2^-25.
decode   a score's fp32 sum over D products is off by at most dS = scale * D *
         2^-24 * sum |q_d k_d| (any order of additions); 2^x by 2^-21; weights
         are rounded (e).  With A = sum_j p_j |c_j|, the numerator is off by
         A (e + dS + 2^-20), the normaliser by (dS + 2^-20) of itself, the
         output by e |out|; dS is small, 2 dS covers the second order:
         A (e + 4 dS + 2^-18) + e |out|.  lse: dS + 2^-20 + |lse| 2^-22.
prefill  as decode; keys and values are rounded to the cache's type on the way:
         dS also takes scale * sum |q_d k_d| * e over the expanded part, and the
         numerator A e once more."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def vk(cuda_ok):
    import vulcan_b200
    vulcan_b200.load()
    return vulcan_b200


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, dtype=torch.float16, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


class Cache:
    """A pool whose sequences own pages in random order; everything that no sequence holds is NaN."""

    def __init__(self, vk, lens, latent=512, rope=64, page=16, dtype=torch.float16, layers=2, layer=1, seed=0, spare=3, first_page=0):
        g = gen(seed)
        self.lens, self.page, self.layer, self.dtype, self.latent, self.rope = list(lens), page, layer, dtype, latent, rope
        need = [-(-n // page) for n in self.lens]
        pages = first_page + sum(need) + spare
        self.pool = vk.LatentKVPool(layers, latent, rope, pages, page_tokens=page, dtype=dtype, zero=False)
        view = self.pool.latent_view()
        view.fill_(float("nan"))
        perm = torch.randperm(pages - first_page, generator=g, device="cuda").add_(first_page).int().cpu()
        self.tables = torch.full((len(self.lens), max(1, max(need, default=1))), -1, dtype=torch.int32)
        self.rows, at = [], 0
        for b, n in enumerate(self.lens):
            ids = perm[at:at + need[b]]
            at += need[b]
            self.tables[b, :need[b]] = ids
            rows = rnd(g, n, latent + rope, dtype=dtype)
            self.rows.append(rows)
            for i, p in enumerate(ids.tolist()):
                part = rows[i * page:(i + 1) * page]
                view[layer, p, :len(part)] = part
        self.tables = self.tables.cuda()
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def check(self):
        torch.cuda.synchronize()
        return self.pool.error_bits()


def decode_bound_check(c, ql, qr, out, lse, scale, tokens, rows=None):
    e = torch.finfo(c.dtype).eps / 2
    d = c.latent + c.rope
    for b, n in enumerate(c.lens):
        x = (c.rows if rows is None else rows)[b].double()
        for t in range(tokens):
            seen = x[:max(0, n - (tokens - 1 - t))]
            o, s = out[b, t].double(), lse[b, t].double()
            if not len(seen):
                assert (o == 0).all() and (s == -float("inf")).all(), (b, t)
                continue
            q = torch.cat([ql[b, t], qr[b, t]], -1).double()
            a = scale * q @ seen.t()
            ds = float((scale * q.abs() @ seen.abs().t()).max()) * d * 2.0 ** -24
            want_lse = torch.logsumexp(a, -1)
            p = torch.exp(a - want_lse[:, None])
            want, size = p @ seen[:, :c.latent], p @ seen[:, :c.latent].abs()
            bound = size * (e + 4 * ds + 2.0 ** -18) + e * want.abs() + 2.0 ** -25
            err = (o - want).abs()
            assert torch.isfinite(err).all(), (b, t)
            assert (err <= bound).all(), "sequence %d token %d: worst %.3g of its bound" % (b, t, (err / bound).max())
            assert ((s - want_lse).abs() <= ds + 2.0 ** -20 + want_lse.abs() * 2.0 ** -22).all(), (b, t)


# ------------------------------------------------------------------ append


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(512, 64, 16), (256, 32, 64), (384, 48, 32), (128, 16, 16)])
@pytest.mark.parametrize("how", ["plain", "norm", "norm+interleaved", "norm+half", "half"])
def test_append(vk, dtype, shape, how):
    """Ragged and uniform chunks; rows written to the right slots, everything else left bit for bit."""
    latent, rope, page = shape
    g = gen(latent + page)
    start, new = [0, 5, 1000, 15, 40], [3, 0, 70, 1, 33]
    c = Cache(vk, [a + n for a, n in zip(start, new)], latent, rope, page, dtype, seed=1)
    before = c.pool.latent_view().clone()
    total = sum(new)
    kv = rnd(g, total + 4, latent + rope, dtype=dtype, std=3.0)  # four rows behind the last sequence
    weight = rnd(g, latent, dtype=dtype) if "norm" in how else None
    rot = vk.RotaryEmbedding(rope, layout="half" if "half" in how else "interleaved") if "half" in how or "inter" in how else None
    offsets = torch.tensor([0] + [sum(new[:i + 1]) for i in range(5)], dtype=torch.int32, device="cuda")
    c.pool.append(1, kv[:, :latent], kv[:, latent:], c.tables, torch.tensor(start, dtype=torch.int32, device="cuda"),
                  offsets=offsets, norm_weight=weight, eps=1e-5, rope=rot)
    assert c.check() == 0
    after, want = c.pool.latent_view(), before.clone()
    e, at = torch.finfo(dtype).eps / 2, 0
    for b in range(5):
        for i in range(new[b]):
            x, pos = kv[at].double(), start[b] + i
            at += 1
            cc, kk, size = x[:latent], x[latent:].clone(), x[latent:].abs()
            if weight is not None:
                cc = cc / torch.sqrt(cc.square().mean() + 1e-5) * weight.double()
            if rot is not None:
                f = torch.tensor(rot.frequencies()[0], dtype=torch.float64, device="cuda") * pos
                ia, ib = (slice(0, rope // 2), slice(rope // 2, rope)) if rot.layout == "half" else (slice(0, rope, 2), slice(1, rope, 2))
                u, w = x[latent:][ia], x[latent:][ib]
                kk[ia], kk[ib] = u * f.cos() - w * f.sin(), u * f.sin() + w * f.cos()
                size = size.clone()
                size[ia] = size[ib] = u.abs() + w.abs()
            row = torch.cat([cc, kk])
            where = (1, int(c.tables[b, pos // page]), pos % page)
            bound = (e + 2.0 ** -19) * row.abs() + 2.0 ** -25
            if rot is not None:
                bound[latent:] += size * 2.0 ** -19
            if weight is None:
                bound[:latent] = 0
            if rot is None:
                bound[latent:] = 0
            err = (after[where].double() - row).abs()
            assert (err <= bound).all(), "%s row %d: worst %.3g of its bound" % (how, at - 1, (err / bound.clamp(min=1e-30)).max())
            want[where] = after[where]
    assert torch.equal(after.view(torch.int16), want.view(torch.int16))
    # the same number for each, without offsets
    kv2 = rnd(g, 10, latent + rope, dtype=dtype)
    c.pool.append(0, kv2[:, :latent], kv2[:, latent:], c.tables, torch.zeros(5, dtype=torch.int32, device="cuda"))
    assert c.check() == 0
    for b in (0, 2, 4):
        assert torch.equal(after[0, int(c.tables[b, 0]), :2], kv2[2 * b:2 * b + 2])


def test_append_many_sequences(vk):
    """More sequences than one round of the offset search, empty ones among them."""
    g, n = gen(3), 1500
    new = torch.randint(0, 3, (n,), generator=g, device="cuda").tolist()
    new[0] = new[-1] = 0
    c = Cache(vk, [max(1, k) for k in new], 128, 16, 16, layers=1, layer=0)
    offsets = torch.tensor([0] + new, device="cuda").cumsum(0).int()
    kv = rnd(g, sum(new), 144)
    c.pool.append(0, kv[:, :128], kv[:, 128:], c.tables, torch.zeros(n, dtype=torch.int32, device="cuda"), offsets=offsets)
    assert c.check() == 0
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(new, device="cuda"))
    slot = torch.arange(len(seq), device="cuda") - offsets[seq]
    assert torch.equal(c.pool.latent_view()[0, c.tables[seq, 0].long(), slot], kv)


def test_append_records_bad_tables(vk):
    """Bad pages and positions are recorded and skipped; the other rows are written."""
    g = gen(4)
    c = Cache(vk, [20, 20, 20, 20], layers=1, layer=0)
    c.tables[1, 1] = c.pool.num_pages
    c.tables[2, 1] = -7
    kv = rnd(g, 4, 576)
    before = c.pool.latent_view().clone()
    pos = torch.tensor([17, 17, 17, 32], dtype=torch.int32, device="cuda")
    c.pool.append(0, kv[:, :512], kv[:, 512:], c.tables, pos)
    assert c.check() == 0x1 | 0x2
    assert torch.equal(c.pool.latent_view()[0, int(c.tables[0, 1]), 1], kv[0])
    before[0, int(c.tables[0, 1]), 1] = kv[0]
    assert torch.equal(c.pool.latent_view().view(torch.int16), before.view(torch.int16))
    c.pool.append(0, kv[:, :512], kv[:, 512:], c.tables, torch.full((4,), -1, dtype=torch.int32, device="cuda"))
    assert c.check() == 0x2
    # offsets that do not ascend reach no memory outside the table
    c.pool.append(0, kv[:, :512], kv[:, 512:], c.tables, torch.full((4,), 1 << 30, dtype=torch.int32, device="cuda"),
                  offsets=torch.tensor([3, -5, 100, 2, 4], dtype=torch.int32, device="cuda"))
    assert c.check() & ~0x3 == 0
    assert torch.equal(c.pool.latent_view().view(torch.int16), before.view(torch.int16))


# ------------------------------------------------------------------ absorbed decode


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(512, 64, 16), (512, 64, 64), (384, 48, 32), (256, 32, 64), (128, 16, 16)])
@pytest.mark.parametrize("rows", [(1, 1), (1, 8), (1, 64), (1, 100), (4, 5), (3, 40)])
def test_decode(vk, dtype, shape, rows):
    """Lengths around the tile and page borders; the rest of the pool is NaN."""
    latent, rope, page = shape
    tokens, heads = rows
    g = gen(latent + heads)
    c = Cache(vk, [1, 0, 63, 64, 65, 2, 128, 700, 16, 17], latent, rope, page, dtype, seed=heads)
    ql, qr = rnd(g, 10, tokens, heads, latent, dtype=dtype, std=0.5), rnd(g, 10, tokens, heads, rope, dtype=dtype)
    out, lse = c.pool.decode(1, ql, qr, c.tables, c.seq_lens, scale=0.07, return_lse=True)
    assert c.check() == 0
    decode_bound_check(c, ql, qr, out, lse, 0.07, tokens)
    again, lse2 = c.pool.decode(1, ql, qr, c.tables, c.seq_lens, scale=0.07, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    if tokens == 1:  # [B, H, latent]
        assert torch.equal(c.pool.decode(1, ql[:, 0], qr[:, 0], c.tables, c.seq_lens, scale=0.07), out[:, 0])


@pytest.mark.parametrize("batch,mean,heads", [(1, 40000, 7), (1, 9000, 64), (3, 5000, 16), (300, 40, 8), (40, 1500, 64)])
def test_decode_splits(vk, batch, mean, heads):
    """One long sequence over all SMs, and more units than SMs."""
    g = gen(batch)
    lens = torch.randint(mean // 2, mean + 1, (batch,), generator=g, device="cuda").tolist()
    c = Cache(vk, lens, page=64 if mean > 5000 else 16, layers=1, layer=0, dtype=torch.bfloat16)
    ql, qr = rnd(g, batch, 1, heads, 512, dtype=torch.bfloat16, std=0.5), rnd(g, batch, 1, heads, 64, dtype=torch.bfloat16)
    out, lse = c.pool.decode(0, ql, qr, c.tables, c.seq_lens, scale=0.07, return_lse=True)
    assert c.check() == 0
    decode_bound_check(c, ql, qr, out, lse, 0.07, 1)


def test_decode_growing_scores(vk):
    """Scores that climb along the keys: the running maximum is rescaled again and again, across CTAs too."""
    g = gen(8)
    c = Cache(vk, [3000], layers=1, layer=0)
    ramp = torch.linspace(0, 60, 3000, device="cuda")[:, None]
    direction = rnd(g, 1, 576).float()
    rows = (direction / direction.norm() * ramp + 0.05 * torch.randn(3000, 576, generator=g, device="cuda")).half()
    view = c.pool.latent_view()
    for i, p in enumerate(c.tables[0].tolist()):
        part = rows[i * 16:(i + 1) * 16]
        view[0, p, :len(part)] = part
    q = (direction * torch.tensor([1.0, -1.0, 0.3, 0.0], device="cuda")[:, None])[None, None].half()  # up, down, slowly, flat
    out, lse = c.pool.decode(0, q[..., :512].contiguous(), q[..., 512:].contiguous(), c.tables, c.seq_lens, scale=0.5, return_lse=True)
    assert c.check() == 0
    decode_bound_check(c, q[..., :512], q[..., 512:], out, lse, 0.5, 1, rows=[rows])


def test_decode_strided_queries(vk):
    """q_latent [H, B, L] from a batched product, q_rope a slice of the projection's heads."""
    g = gen(11)
    c = Cache(vk, [100, 37, 64])
    ql = rnd(g, 20, 3, 512, std=0.5).transpose(0, 1)
    qr = rnd(g, 3, 20, 192)[..., 128:]
    out, lse = c.pool.decode(1, ql, qr, c.tables, c.seq_lens, scale=0.07, return_lse=True)
    assert c.check() == 0
    decode_bound_check(c, ql[:, None], qr[:, None], out[:, None], lse[:, None], 0.07, 1)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_decode_non_finite_draft(vk, bad):
    """A drafted token's broken row reaches the tokens that see it, and no other."""
    g = gen(12)
    c = Cache(vk, [65, 130], layers=1, layer=0)
    tokens = 3
    ql, qr = rnd(g, 2, tokens, 4, 512, std=0.5), rnd(g, 2, tokens, 4, 64)
    rows = []
    for b, n in enumerate(c.lens):  # the last of the three new rows
        c.pool.latent_view()[0, int(c.tables[b, (n - 1) // 16]), (n - 1) % 16, 100] = bad
        rows.append(c.rows[b])
    out, lse = c.pool.decode(0, ql, qr, c.tables, c.seq_lens, scale=0.07, return_lse=True)
    assert c.check() == 0
    c2 = type("C", (), dict(dtype=c.dtype, latent=512, rope=64, lens=c.lens, rows=rows))
    # tokens 0 and 1 do not see it
    short = type("C", (), dict(vars(c2), lens=[n - 1 for n in c.lens]))
    decode_bound_check(short, ql[:, :2], qr[:, :2], out[:, :2], lse[:, :2], 0.07, 2)
    if bad != bad:
        assert torch.isnan(out[:, 2]).all()


def test_decode_records_bad_lengths_and_pages(vk):
    g = gen(13)
    c = Cache(vk, [50, 60, 70, 80])
    lens = c.seq_lens.clone()
    lens[1], lens[2] = -3, c.tables.shape[1] * 16 + 1
    ql, qr = rnd(g, 4, 1, 8, 512, std=0.5), rnd(g, 4, 1, 8, 64)
    out, lse = c.pool.decode(1, ql, qr, c.tables, lens, scale=0.07, return_lse=True)
    assert c.check() == 0x4
    c.lens = [50, 0, 0, 80]
    decode_bound_check(c, ql, qr, out, lse, 0.07, 1)
    tables = c.tables.clone()
    tables[3, 2] = c.pool.num_pages + 5
    out = c.pool.decode(1, ql, qr, tables, torch.tensor([50, 0, 0, 80], dtype=torch.int32, device="cuda"), scale=0.07)
    assert c.check() == 0x1
    c.lens = [50]
    decode_bound_check(c, ql[:1], qr[:1], out[:1], lse[:1], 0.07, 1)


def test_decode_graph_streams_and_workspace(vk):
    """A captured call replays with other lengths; two calls run side by side; a dirty workspace does not matter."""
    g = gen(14)
    c = Cache(vk, [500, 33, 1000])
    ql, qr = rnd(g, 3, 1, 16, 512, std=0.5), rnd(g, 3, 1, 16, 64)
    size = c.pool.decode_workspace_size(3, 1, 16)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN patterns
    out, lse = torch.empty(3, 1, 16, 512, device="cuda").half(), torch.empty(3, 1, 16, device="cuda")
    lens = c.seq_lens.clone()
    graph = torch.cuda.CUDAGraph()
    c.pool.decode(1, ql, qr, c.tables, lens, 0.07, out=out, lse=lse, workspace=ws)
    with torch.cuda.graph(graph):
        c.pool.decode(1, ql, qr, c.tables, lens, 0.07, out=out, lse=lse, workspace=ws)
    for new in ([500, 33, 1000], [1, 0, 64], [499, 20, 641], [0, 0, 0]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        out.fill_(5)
        graph.replay()
        assert c.check() == 0
        c.lens = new
        decode_bound_check(c, ql, qr, out, lse, 0.07, 1)
    c.lens = [500, 33, 1000]
    want = c.pool.decode(1, ql, qr, c.tables, c.seq_lens, 0.07)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            got.append(c.pool.decode(1, ql, qr, c.tables, c.seq_lens, 0.07, stream=s))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_rows_beyond_four_gigabytes(vk):
    """Pages whose bytes and elements lie past 2^32: append, decode and prefill."""
    g = gen(15)
    first = (5 << 30) // (64 * 576 * 2)
    c = Cache(vk, [300, 129], page=64, layers=1, layer=0, first_page=first, seed=2)
    kv = rnd(g, 2, 576)
    c.pool.append(0, kv[:, :512], kv[:, 512:], c.tables, c.seq_lens - 1)
    c.rows[0][-1], c.rows[1][-1] = kv[0], kv[1]
    ql, qr = rnd(g, 2, 1, 4, 512, std=0.5), rnd(g, 2, 1, 4, 64)
    out, lse = c.pool.decode(0, ql, qr, c.tables, c.seq_lens, 0.07, return_lse=True)
    assert c.check() == 0
    decode_bound_check(c, ql, qr, out, lse, 0.07, 1)
    prefill_check(c, g, [20, 129], 2)


# ------------------------------------------------------------------ expanded prefill


def prefill_check(c, g, new, heads, scale=0.0, extra=0, **kw):
    """Runs the last new[b] rows of each sequence as a chunk and holds every row to its bound."""
    layer, total = c.layer, sum(new)
    q = rnd(g, total + extra, heads, 128 + c.rope, dtype=c.dtype)
    w = rnd(g, heads * 256, c.latent, dtype=c.dtype, std=c.latent ** -0.5)
    offsets = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device="cuda")
    out = torch.full((total + extra, heads, 128), 9.0, device="cuda").to(c.dtype)
    got = c.pool.prefill(layer, q, w, c.tables, c.seq_lens - torch.tensor(new, dtype=torch.int32, device="cuda"), offsets=offsets,
                         out=out, scale=scale, **kw)
    assert got is out and c.check() == 0
    assert (out[total:] == 9).all()  # rows behind the last sequence
    sc = scale or (128 + c.rope) ** -0.5
    e, at = torch.finfo(c.dtype).eps / 2, 0
    for b, n in enumerate(new):
        if not n:
            continue
        x = c.rows[b].double()
        hidden = torch.arange(c.lens[b], device="cuda")[None] > torch.arange(c.lens[b] - n, c.lens[b], device="cuda")[:, None]
        for h in range(heads):
            up = w[h * 256:(h + 1) * 256].double()
            kv = x[:, :c.latent] @ up.t()
            k, v = torch.cat([kv[:, :128], x[:, c.latent:]], -1), kv[:, 128:]
            qq = q[at:at + n, h].double()
            a = (sc * qq @ k.t()).masked_fill(hidden, -float("inf"))
            exp_part = sc * qq[:, :128].abs() @ k[:, :128].abs().t()
            ds = (exp_part * e + sc * (qq.abs() @ k.abs().t()) * (128 + c.rope) * 2.0 ** -24).masked_fill(hidden, 0).amax(-1, keepdim=True)
            # the expansion's own fp32 sums, as a share of |W| |c|
            ds = ds + (sc * qq[:, :128].abs() @ (x[:, :c.latent].abs() @ up[:128].abs().t()).t()).masked_fill(hidden, 0).amax(-1, keepdim=True) * c.latent * 2.0 ** -24
            p = torch.softmax(a, -1)
            want, size = p @ v, p @ v.abs()
            grow = torch.expm1(2 * ds)
            bound = size * (2 * e + e * e + grow + 2.0 ** -18) + e * want.abs() + 2.0 ** -25 + p @ (x[:, :c.latent].abs() @ up[128:].abs().t()) * c.latent * 2.0 ** -24
            err = (out[at:at + n, h].double() - want).abs()
            assert torch.isfinite(err).all(), (b, h)
            assert (err <= bound).all(), "sequence %d head %d: worst %.3g of its bound" % (b, h, (err / bound).max())
        at += n
    return q, w, out, offsets


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(512, 64, 16), (384, 48, 32), (256, 32, 64), (128, 16, 16)])
@pytest.mark.parametrize("heads", [1, 3])
def test_prefill(vk, dtype, shape, heads):
    """Ragged chunks with and without a prefix, borders of the row and key tiles, empty chunks, rows behind the end."""
    g = gen(shape[0] + heads)
    c = Cache(vk, [1, 300, 128, 0, 257, 640, 500, 129, 5], *shape, dtype, seed=heads)
    prefill_check(c, g, [1, 300, 1, 0, 129, 256, 0, 129, 2], heads, extra=3)


def test_prefill_one_chunk_each_and_default_bounds(vk):
    g = gen(21)
    c = Cache(vk, [200, 100])
    q = rnd(g, 2, 40, 5, 192)
    w = rnd(g, 5 * 256, 512, std=512 ** -0.5)
    pos = c.seq_lens - 40
    got = c.pool.prefill(1, q, w, c.tables, pos)
    assert got.shape == (2, 40, 5, 128)
    offsets = torch.tensor([0, 40, 80], dtype=torch.int32, device="cuda")
    flat = c.pool.prefill(1, q.view(80, 5, 192), w, c.tables, pos, offsets=offsets, max_tokens=40, max_seq_len=200)
    assert c.check() == 0
    assert torch.equal(got.view(80, 5, 128), flat)
    # strided queries and a weight cut from a wider one
    wide = torch.cat([w, w], 1)[:, :512]
    qs = torch.cat([q.view(80, 5, 192)] * 2, -1)[..., :192]
    assert torch.equal(c.pool.prefill(1, qs, wide, c.tables, pos, offsets=offsets, max_tokens=40, max_seq_len=200), flat)


@pytest.mark.parametrize("new,prefix,heads,batch", [(1, 3000, 2, 1), (200, 5000, 4, 1), (257, 2000, 1, 2), (33, 900, 3, 2)])
def test_prefill_cut_along_keys(vk, new, prefix, heads, batch):
    """Few query tiles behind long prefixes: each is cut into key ranges, some of which a row does not see."""
    g = gen(prefix)
    lens = [prefix + new, prefix // 3 + new][:batch]
    c = Cache(vk, lens, layers=1, layer=0, dtype=torch.bfloat16)
    prefill_check(c, g, [new, max(1, new // 2)][:batch], heads, scale=0.05)


def test_prefill_graph_and_streams(vk):
    """Append and prefill captured together replay with other chunks; calls on several streams run side by side."""
    g = gen(41)
    c = Cache(vk, [400, 700, 90], seed=3)
    total, heads = 330, 4
    q, w = rnd(g, total, heads, 192), rnd(g, heads * 256, 512, std=512 ** -0.5)
    lat, kr = rnd(g, total, 512), rnd(g, total, 64)
    pos, offsets = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")

    def chunk(new):
        offsets.copy_(torch.tensor([0, new[0], new[0] + new[1], sum(new)], dtype=torch.int32))
        pos.copy_(c.seq_lens - torch.tensor(new, dtype=torch.int32, device="cuda"))

    def run(out, stream=None):
        c.pool.append(1, lat, kr, c.tables, pos, offsets=offsets, stream=stream)
        return c.pool.prefill(1, q, w, c.tables, pos, offsets=offsets, max_tokens=200, max_seq_len=704, out=out, stream=stream)

    out = torch.empty(total, heads, 128, device="cuda").half()
    chunk([10, 20, 30])
    run(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out)
    for new in ([100, 200, 30], [1, 0, 90], [0, 0, 0], [17, 129, 1]):
        chunk(new)
        want = run(torch.full_like(out, 4))
        out.fill_(4)
        graph.replay()
        assert c.check() == 0
        assert torch.equal(out, want), new
        assert (out[sum(new):] == 4).all()
    chunk([100, 200, 30])
    want = run(torch.empty_like(out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [c.pool.prefill(1, q, w, c.tables, pos, offsets=offsets, max_tokens=200, max_seq_len=704, stream=s)
           for _ in range(3) for s in streams]
    torch.cuda.synchronize()
    assert c.check() == 0
    assert all(torch.equal(x, want) for x in got)


def test_prefill_head_groups(vk):
    """A bound on the lengths that makes the workspace hold a part of the heads at a time."""
    g = gen(23)
    c = Cache(vk, [150], 128, 16, 64, layers=1, layer=0)
    c.tables = torch.cat([c.tables, torch.full((1, 1600), -1, dtype=torch.int32, device="cuda")], 1)
    bound = 100000  # 100096 rows of 512 bytes a head: 20 heads a GiB, 7 a group of 20
    assert c.pool.prefill_workspace_size(1, bound, 41) < 100096 * 512 * 41
    prefill_check(c, g, [150], 41, max_tokens=150, max_seq_len=bound)


def test_prefill_non_finite_latents(vk):
    """A chunk token with a broken latent reaches the rows that see it, and no earlier ones."""
    for bad in (float("nan"), float("inf")):
        g = gen(24)
        c = Cache(vk, [100], layers=1, layer=0)
        q, w = rnd(g, 100, 2, 192), rnd(g, 512, 512, std=512 ** -0.5)
        pos = torch.zeros(1, dtype=torch.int32, device="cuda")
        want = c.pool.prefill(0, q, w, c.tables, pos)
        c.pool.latent_view()[0, int(c.tables[0, 70 // 16]), 70 % 16, 3] = bad
        got = c.pool.prefill(0, q, w, c.tables, pos)
        assert c.check() == 0
        assert torch.equal(got[:70], want[:70])
        assert torch.isnan(got[70:]).all()


def test_prefill_values_beyond_the_type(vk):
    """A finite latent whose value overflows fp16 leaves the rows that may not see it as they were."""
    g = gen(25)
    c = Cache(vk, [100], layers=1, layer=0)
    q, w = rnd(g, 100, 2, 192), rnd(g, 512, 512, std=512 ** -0.5)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = c.pool.prefill(0, q, w, c.tables, pos)
    row = 6000 * torch.sign(w[128])  # the first value element of head 0
    assert float((row.double() * w[128].double()).sum()) > 70000
    assert float((w[:128].double() @ row.double()).abs().max()) < 60000
    c.pool.latent_view()[0, int(c.tables[0, 70 // 16]), 70 % 16, :512] = row
    got = c.pool.prefill(0, q, w, c.tables, pos)
    assert c.check() == 0
    assert torch.equal(got[:70], want[:70])
    assert torch.isfinite(got).all()


def test_prefill_records_what_is_out_of_bounds(vk):
    """Sequences beyond the given bounds are recorded and left out; the others are computed."""
    g = gen(25)
    c = Cache(vk, [90, 90, 90])
    q, w = rnd(g, 90, 2, 192), rnd(g, 512, 512, std=512 ** -0.5)
    offsets = torch.tensor([0, 30, 60, 90], dtype=torch.int32, device="cuda")
    pos = torch.full((3,), 60, dtype=torch.int32, device="cuda")
    want = c.pool.prefill(1, q, w, c.tables, pos, offsets=offsets, max_tokens=30, max_seq_len=90)
    assert c.check() == 0

    def others(bit, keep, **kw):
        out = torch.full_like(want, 3.0)
        args = dict(dict(offsets=offsets, max_tokens=30, max_seq_len=90, out=out), **kw)
        c.pool.prefill(1, q, w, args.pop("tables", c.tables), args.pop("pos", pos), **args)
        assert c.check() == bit
        for b in range(3):
            part = out[30 * b:30 * b + 30]
            assert torch.equal(part, want[30 * b:30 * b + 30]) if b in keep else b in (1,)
        return out

    far, neg = pos.clone(), pos.clone()
    far[1], neg[1] = 61, -1
    assert (others(0x4, (0, 2), pos=far)[30:60] == 3).all()
    assert (others(0x4, (0, 2), pos=neg)[30:60] == 3).all()
    tables = c.tables.clone()
    tables[1, 1] = -1
    others(0x1, (0, 2), tables=tables)
    out = torch.full_like(want, 3.0)
    c.pool.prefill(1, q, w, c.tables, pos, offsets=torch.tensor([0, 30, 95, 90], dtype=torch.int32, device="cuda"), max_tokens=70,
                   max_seq_len=90, out=out)
    assert c.check() == 0x4
    assert torch.equal(out[:30], want[:30]) and (out[30:] == 3).all()


def test_nothing_to_do(vk):
    """No sequences, no tokens, no rows: nothing is launched or written."""
    c = Cache(vk, [40])
    kv = rnd(gen(30), 2, 576)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    c.pool.append(0, kv[:0, :512], kv[:0, 512:], c.tables, c.seq_lens)
    c.pool.append(0, kv[:0, :512], kv[:0, 512:], c.tables[:0], none)
    out, lse = c.pool.decode(0, torch.empty(0, 4, 512, device="cuda").half(), torch.empty(0, 4, 64, device="cuda").half(), c.tables[:0], none,
                             0.1, return_lse=True)
    assert out.shape == (0, 4, 512) and lse.shape == (0, 4)
    assert c.pool.prefill(0, torch.empty(0, 2, 192, device="cuda").half(), rnd(gen(1), 512, 512), c.tables, c.seq_lens).shape == (0, 2, 128)
    assert c.check() == 0


# ------------------------------------------------------------------ refusals


def test_refusals(vk):
    g = gen(31)
    c = Cache(vk, [40, 40])
    pool, t, n = c.pool, c.tables, c.seq_lens
    kv = rnd(g, 4, 576)
    ql, qr = rnd(g, 2, 1, 4, 512), rnd(g, 2, 1, 4, 64)
    q, w = rnd(g, 4, 4, 192), rnd(g, 1024, 512)
    lib, K = pool._lib, vk.VKError
    closed = vk.RotaryEmbedding(64)
    closed.close()
    for call in (lambda: pool.append(2, kv[:, :512], kv[:, 512:], t, n), lambda: pool.decode(-1, ql, qr, t, n, 0.1),
                 lambda: pool.prefill(2, q, w, t, n - 2),
                 lambda: pool.append(0, kv[:3, :512], kv[:3, 512:], t, n),           # 3 rows of 2 sequences
                 lambda: pool.append(0, kv.view(-1)[4:4 + 3 * 512].view(3, 512)[:2], kv[:2, 512:], t, n),  # 8-byte aligned
                 lambda: pool.append(0, kv[:, :512], kv[:, 512:], t, n, norm_weight=kv[0, :512].clone(), eps=-1.0),
                 lambda: pool.append(0, kv[:, :512], kv[:, 512:], t, n, rope=vk.RotaryEmbedding(32)),
                 lambda: pool.decode(0, ql, qr, t, n, 0.0), lambda: pool.decode(0, ql, qr, t, n, float("nan")),
                 lambda: pool.decode(0, ql, qr, t, n, 0.1, workspace=torch.empty(100, dtype=torch.uint8, device="cuda")),
                 lambda: pool.decode(0, ql, rnd(g, 2, 1, 4, 68)[..., 2:66], t, n, 0.1),  # strides of 68
                 lambda: pool.prefill(0, q, w, t, n - 2, scale=-1.0),
                 lambda: pool.prefill(0, q, w, t, n - 2, max_tokens=1), lambda: pool.prefill(0, q, w, t, n - 2, max_seq_len=1),
                 lambda: pool.prefill(0, q, w, t, n - 2, max_seq_len=10000),
                 lambda: pool.prefill(0, q, w, t, n - 2, workspace=torch.empty(100, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(K):
            call()
    for call in (lambda: pool.append(0, kv[:, :500], kv[:, 512:], t, n), lambda: pool.append(0, kv[:, :512], kv[:3, 512:], t, n),
                 lambda: pool.append(0, kv[:, :512], kv[:, 512:], t, n[:1]), lambda: pool.append(0, kv[:, :512], kv[:, 512:], t[0], n),
                 lambda: pool.decode(0, ql[..., :256], qr, t, n, 0.1), lambda: pool.decode(0, ql, qr[:, :, :3], t, n, 0.1),
                 lambda: pool.decode(0, ql[:1], qr[:1], t, n, 0.1), lambda: pool.decode(0, ql.cpu(), qr, t, n, 0.1),
                 lambda: pool.decode(0, ql, qr, t, n, 0.1, out=torch.empty(2, 1, 4, 256, device="cuda").half()),
                 lambda: pool.prefill(0, q[..., :128], w, t, n), lambda: pool.prefill(0, q, w[:512], t, n),
                 lambda: pool.prefill(0, q, w, t, n, offsets=n),
                 lambda: pool.decode(0, ql, qr, t, n, 0.1, workspace=torch.empty(1 << 27, dtype=torch.uint8)),
                 lambda: pool.append(0, kv[:, :512], kv[:, 512:], t, n, rope=closed)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: pool.append(0, kv[:, :512].float(), kv[:, 512:], t, n), lambda: pool.decode(0, ql.bfloat16(), qr, t, n, 0.1),
                 lambda: pool.decode(0, ql, qr, t.long(), n, 0.1), lambda: pool.prefill(0, q, w.bfloat16(), t, n),
                 lambda: pool.plan([1, 2], 4), lambda: pool.set_rope(10000.0)):
        with pytest.raises(TypeError):
            call()
    # the entry points of K/V pages refuse a latent pool, and these refuse a K/V pool
    kvp = vk.PagedKVPool(1, 1, 128, 4)
    import ctypes
    p = ctypes.c_void_p
    assert lib.vk_append(pool.handle, 0, p(kv.data_ptr()), p(kv.data_ptr()), p(t.data_ptr()), 1, p(n.data_ptr()), 1, 1, None) == 7
    assert lib.vk_decode(pool.handle, 0, p(ql.data_ptr()), p(ql.data_ptr()), p(t.data_ptr()), 1, p(n.data_ptr()), 1, 1, 16, 0.0, None, 0, None) == 7
    assert lib.vk_prefill(pool.handle, 0, p(ql.data_ptr()), p(ql.data_ptr()), p(t.data_ptr()), 1, p(n.data_ptr()), 1, 1, 1, 0.0, None) == 7
    assert lib.vk_set_rope(pool.handle, 10000.0) == 7
    assert lib.vk_latent_append(kvp.handle, 0, kv.data_ptr(), 576, kv.data_ptr(), 576, None, 0.0, None, t.data_ptr(), 1, n.data_ptr(), None, 1, 1, None) == 7
    assert lib.vk_latent_decode_workspace_size(kvp.handle, 1, 1, 1) == 0
    assert lib.vk_pool_kv_format(pool.handle) == 2
    assert c.check() == 0


# ------------------------------------------------------------------ pages, and a run together


@pytest.mark.parametrize("own_memory", [False, True])
def test_page_operations(vk, own_memory):
    """Fork by copy, compaction with remapped tables, swap out and in: rows survive bit for bit."""
    g = gen(41)
    pool = vk.LatentKVPool(3, 256, 32, 12, page_tokens=32, dtype=torch.bfloat16, own_memory=own_memory)
    ids = pool.alloc(6)
    pool.free(ids[:3])
    ids = ids[3:]
    t = torch.tensor([ids], dtype=torch.int32, device="cuda")
    n = torch.tensor([90], dtype=torch.int32, device="cuda")
    for layer in range(3):
        kv = rnd(g, 90, 288, dtype=torch.bfloat16)
        pool.append(layer, kv[:, :256], kv[:, 256:], t, n - 90)
    ql, qr = rnd(g, 1, 8, 256, dtype=torch.bfloat16), rnd(g, 1, 8, 32, dtype=torch.bfloat16)
    want = [pool.decode(layer, ql, qr, t, n, 0.1) for layer in range(3)]
    same = lambda tab: all(torch.equal(pool.decode(layer, ql, qr, tab, n, 0.1), want[layer]) for layer in range(3))  # noqa: E731
    fork = pool.alloc(3)
    tf = torch.tensor([fork], dtype=torch.int32, device="cuda")
    pool.copy_pages(t[0].contiguous(), tf[0].contiguous())
    assert same(tf)
    src, dst = pool.compact_plan()
    page_map = torch.arange(12, dtype=torch.int32, device="cuda")
    if src:
        page_map[torch.tensor(src, device="cuda")] = torch.tensor(dst, dtype=torch.int32, device="cuda")
        pool.copy_pages(torch.tensor(src, dtype=torch.int32, device="cuda"), torch.tensor(dst, dtype=torch.int32, device="cuda"))
        vk.remap_block_tables(t, page_map)
        vk.remap_block_tables(tf, page_map)
    assert sorted(t[0].tolist() + tf[0].tolist()) == list(range(6)) and same(t) and same(tf)
    host = torch.empty(3 * pool.page_bytes, dtype=torch.uint8, pin_memory=True)
    pool.swap_out(t[0].tolist(), host)
    torch.cuda.synchronize()
    back = pool.swap_in(host, 3)
    torch.cuda.synchronize()
    assert same(torch.tensor([back], dtype=torch.int32, device="cuda")) and same(tf)
    assert pool.error_bits() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_layer_serves(vk, dtype):
    """A layer as it is served: a prompt's chunk, a second chunk behind it, then single and drafted tokens in the
    absorbed form, all against one attention in 64 bits over the whole sequence, rows made from the inputs.

    Bound: the cache's rows carry one rounding (e of each element), which moves a score by at most
    scale * sum |q||k| * e * 2 (queries are rounded after their rotation too) and a value by e: with the paths'
    own roundings, |out - want| <= A (6 e + 2 (exp(2 dS) - 1)) for dS = scale * sum |q||k| * 4 e."""
    g, heads, latent, rope, batch = gen(51), 6, 512, 64, 2
    e, scale = torch.finfo(dtype).eps / 2, (128 + rope) ** -0.5
    steps = [150, 70, 1, 1, 3]  # prompt chunk, chunk, token, token, three drafted
    total = sum(steps)
    pool = vk.LatentKVPool(1, latent, rope, 40, dtype=dtype)
    tables = torch.tensor([pool.alloc(15) for _ in range(batch)], dtype=torch.int32, device="cuda")
    rotary = vk.RotaryEmbedding(rope, layout="interleaved", scaling="linear", factor=2.0)
    weight = 1 + rnd(g, latent, dtype=dtype, std=0.1)
    w = rnd(g, heads * 256, latent, dtype=dtype, std=latent ** -0.5)
    up = w.view(heads, 256, latent)
    kv = rnd(g, batch, total, latent + rope, dtype=dtype)
    q = rnd(g, batch, total, heads, 128 + rope, dtype=dtype)

    # 64 bits
    f = torch.tensor(rotary.frequencies()[0], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones(total, rope // 2, dtype=torch.float64, device="cuda"),
                       torch.arange(total, device="cuda").double()[:, None] * f)

    def rotate(x):  # [..., total, (heads,) rope]
        z = torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous())
        return torch.view_as_real(z * (turn if x.dim() == 3 else turn[:, None])).flatten(-2)

    c = kv[..., :latent].double()
    c = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + 1e-6) * weight.double()
    kr, qr = rotate(kv[..., latent:]), rotate(q[..., 128:])
    keys = torch.einsum("bkc,hdc->bhkd", c, up[:, :128].double())
    vals = torch.einsum("bkc,hdc->bhkd", c, up[:, 128:].double())
    s = torch.einsum("bthd,bhkd->bhtk", q[..., :128].double(), keys) + torch.einsum("bthd,bkd->bhtk", qr, kr)
    hidden = torch.ones(total, total, device="cuda").triu(1).bool()
    p = torch.softmax((s * scale).masked_fill(hidden, -float("inf")), -1)
    want, size = torch.einsum("bhtk,bhkd->bthd", p, vals), torch.einsum("bhtk,bhkd->bthd", p, vals.abs())
    # |q| |k| with the latent's own absolute values: the absorbed form sums over them
    big = torch.einsum("bthd,bhkd->bhtk", q[..., :128].abs().double(), torch.einsum("bkc,hdc->bhkd", c.abs(), up[:, :128].abs().double()))
    ds = (scale * (big + torch.einsum("bthd,bkd->bhtk", qr.abs(), kr.abs()))).masked_fill(hidden, 0).amax(-1) * 4 * e
    rough = torch.einsum("bhtk,bhkd->bthd", p, torch.einsum("bkc,hdc->bhkd", c.abs(), up[:, 128:].abs().double()))
    bound = rough * (6 * e + 2 * torch.expm1(2 * ds).transpose(1, 2)[..., None]) + size * 6 * e

    at = 0
    for n in steps:
        now = slice(at, at + n)
        pos = torch.full((batch,), at, dtype=torch.int32, device="cuda")
        rows = kv[:, now].reshape(batch * n, latent + rope)
        qn = q[:, now].clone()
        token_pos = (torch.arange(at, at + n, device="cuda").int().repeat(batch)).contiguous()
        rotary.apply(qn[..., 128:], token_pos, out=qn[..., 128:])
        pool.append(0, rows[:, :latent], rows[:, latent:], tables, pos, norm_weight=weight, eps=1e-6, rope=rotary)
        if n > 10:
            out = pool.prefill(0, qn, w, tables, pos, max_seq_len=at + n)
        else:
            ql = torch.einsum("bthd,hdc->bthc", qn[..., :128].float(), up[:, :128].float()).to(dtype)
            lat = pool.decode(0, ql, qn[..., 128:], tables, pos + n, scale)
            out = torch.einsum("bthc,hdc->bthd", lat.float(), up[:, 128:].float())
        torch.cuda.synchronize()
        assert pool.error_bits() == 0
        err = (out.double() - want[:, now]).abs()
        assert (err <= bound[:, now]).all(), "tokens %d..: worst %.3g of its bound" % (at, (err / bound[:, now]).max())
        # far inside the bound on average: a wrong row or mask would not be
        assert float(err.norm() / want[:, now].norm()) < 8 * e
        at += n


def test_scheduler_over_a_latent_pool(vk):
    """Sequences admitted, grown, evicted to the host, restored and compacted keep their rows: each decode equals one over
    rows kept aside."""
    from vulcan_b200.scheduler import PagedKVScheduler
    g, page = gen(61), 64
    pool = vk.LatentKVPool(1, 256, 32, 9, page_tokens=page)
    host = torch.empty(8 * pool.page_bytes, dtype=torch.uint8).pin_memory()
    sched = PagedKVScheduler(pool, host, 8)
    rows = {}

    def tables(ids):
        return torch.from_numpy(sched.block_table(ids)).cuda(), torch.from_numpy(sched.lengths(ids)).cuda()

    def append(sid, n):
        new = rnd(g, n, 288)
        bt, _ = tables([sid])
        at = 0 if sid not in rows else len(rows[sid])
        rows[sid] = new if not at else torch.cat([rows[sid], new])
        pool.append(0, new[:, :256], new[:, 256:], bt, torch.tensor([at], dtype=torch.int32, device="cuda"))

    def check(ids):
        bt, lens = tables(ids)
        ql, qr = rnd(g, len(ids), 4, 256), rnd(g, len(ids), 4, 32)
        out, lse = pool.decode(0, ql, qr, bt, lens, 0.06, return_lse=True)
        torch.cuda.synchronize()
        assert pool.error_bits() == 0
        c = type("Rows", (), dict(lens=[len(rows[i]) for i in ids], rows=[rows[i] for i in ids], dtype=torch.float16, latent=256, rope=32))
        decode_bound_check(c, ql[:, None], qr[:, None], out[:, None], lse[:, None], 0.06, 1)

    for sid, n in ((0, 130), (1, 64), (2, 190)):
        assert sched.admit(sid, n)
        append(sid, n)
    assert [len(sched.seqs[i].pages) for i in range(3)] == [3, 1, 3]
    check([0, 1, 2])
    assert sched.grow(1)
    append(1, 1)
    assert sched.evict(0)
    assert sched.admit(3, 200)  # pages that were sequence 0's
    append(3, 200)
    check([1, 2, 3])
    torch.cuda.synchronize()
    sched.release(2)
    ids = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    assert sched.compact(lambda src, dst: pool.copy_pages(ids(src), ids(dst))) > 0
    check([3, 1])
    assert sched.restore(0)
    torch.cuda.synchronize()
    check([3, 0, 1])
