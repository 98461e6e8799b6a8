"""GPU tests of the latent cache's attention where its arithmetic is tight, against 64 bits.

Tolerances as in test_gpu_latent.py, and for fp16 weights one more term: a weight is
stored as 2^7 (up to 2^15) times its share of the row's largest, so that one below 2^-21
of the largest lies among fp16's subnormals and is off by up to 2^-25 / 2^7 = 2^-32 of the
largest weight p_max: p_max 2^-32 sum_j |v_j| in all.  Over 131,072 keys the products' sum,
one fp32 addition for 16 keys whose result may be cut instead of rounded (2^-23 of it), counts
too: sum_j p_j |v_j| * keys / 16 * 2^-23."""
import math

import pytest
import torch

from .test_gpu_latent import Cache, decode_bound_check, gen, prefill_check, rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vk(cuda_ok):
    import vulcan_b200
    vulcan_b200.load()
    return vulcan_b200


# ------------------------------------------------------------------ one dominant key

BITS = [0.0, 12.0, 20.0, 24.0, 25.0, 26.0, 28.0, 34.0]  # binary orders between the dominant key and the others
KEYS = 131072


def sink(vk, at, dtype=torch.float16):
    """A sequence whose key `at` is the only one with a score, the others hold the values."""
    g = gen(at)
    c = Cache(vk, [KEYS], 128, 16, 64, layers=1, layer=0, dtype=dtype)
    rows = torch.cat([0.5 + torch.rand(KEYS, 128, generator=g, device="cuda"), torch.zeros(KEYS, 16, device="cuda")], -1).to(dtype)
    rows[:, 0] = 0
    rows[at] = 0
    rows[at, 0] = 16
    c.pool.latent_view()[0, c.tables[0].long()] = rows.view(-1, 64, 144)
    return c, rows


def weak_weight_bound(p, v, e, share):
    """Bound of sum_j p_j v_j without the output's own rounding; `share`: roundings of a product's factors."""
    share = share + v.shape[0] / 16 * 2.0 ** -23
    return p @ v.abs() * share + p.amax(-1, keepdim=True) * 2.0 ** -32 * v.abs().sum(0) * (e < 2.0 ** -9)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("at,sequences", [(5, 1), (KEYS - 70, 1), (5, 200)])
def test_decode_one_dominant_key(vk, dtype, at, sequences):
    """Many keys of little weight each keep their part of the output.  200 sequences that share their pages: a CTA has
    whole sequences to itself, and the dominant key stands against all the others in it."""
    c, rows = sink(vk, at, dtype)
    scale, e = 0.07, torch.finfo(dtype).eps / 2
    ql = torch.zeros(sequences, len(BITS), 128, device="cuda")
    ql[..., 0] = torch.tensor(BITS, device="cuda") * math.log(2) / (16 * scale)
    ql = ql.to(dtype)
    qr = torch.zeros(sequences, len(BITS), 16, device="cuda").to(dtype)
    tables = c.tables.expand(sequences, -1).contiguous()
    lens = torch.full((sequences,), KEYS, dtype=torch.int32, device="cuda")
    out, lse = c.pool.decode(0, ql, qr, tables, lens, scale, return_lse=True)
    assert c.check() == 0
    x = rows.double()
    a = scale * ql[0].double() @ x[:, :128].t()
    want_lse = torch.logsumexp(a, -1)
    p = torch.exp(a - want_lse[:, None])
    want = p @ x[:, :128]
    ds = a.abs().amax(-1, keepdim=True) * 144 * 2.0 ** -24
    bound = weak_weight_bound(p, x[:, :128], e, e + 4 * ds + 2.0 ** -18) + e * want.abs() + 2.0 ** -25
    err = (out.double() - want).abs()
    assert (err <= bound).all(), "rows' worst %s of the bound" % (err / bound).amax((0, 2)).tolist()
    assert ((lse.double() - want_lse).abs() <= ds[:, 0] + 2.0 ** -20 + want_lse.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("at,heads", [(5, 2), (KEYS - 70, 2), (5, 40)])
def test_prefill_one_dominant_key(vk, dtype, at, heads):
    """As above in the expanded form: keys [c_0, 0, ...] (exact in 16 bits), values c; few heads cut along the keys, and many."""
    c, rows = sink(vk, at, dtype)
    scale, e, new = 0.07, torch.finfo(dtype).eps / 2, len(BITS)
    w = torch.zeros(heads, 256, 128, device="cuda")
    w[:, 0, 0] = 1
    w[:, 128:] = torch.eye(128, device="cuda")
    w = w.view(heads * 256, 128).to(dtype)
    q = torch.zeros(new, heads, 144, device="cuda")
    q[..., 0] = (torch.tensor(BITS, device="cuda") * math.log(2) / (16 * scale))[:, None]
    q = q.to(dtype)
    out = c.pool.prefill(0, q, w, c.tables, c.seq_lens - new, scale=scale)
    assert c.check() == 0
    x = rows[:, :128].double()
    hidden = torch.arange(KEYS, device="cuda")[None] > torch.arange(KEYS - new, KEYS, device="cuda")[:, None]
    a = scale * q[:, 0, :1].double() @ x[:, :1].t()
    p = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
    want = p @ x
    ds = a.abs().amax(-1, keepdim=True) * (144 + 128) * 2.0 ** -24
    # values are exact: c times one
    bound = weak_weight_bound(p, x, e, e + 4 * ds + 2.0 ** -18) + e * want.abs() + 2.0 ** -25
    err = (out.double() - want[:, None]).abs()
    assert (err <= bound[:, None]).all(), "rows' worst %s of the bound" % (err / bound[:, None]).amax((1, 2)).tolist()


# ------------------------------------------------------------------ infinite and NaN latents


def decode_pattern_check(c, rows, ql, qr, out, lse, scale):
    """Every row against the formula in 64 bits: a weight of zero times an infinite element is NaN in that element, an
    infinite or NaN score makes the row NaN; finite elements are held to the usual bound."""
    e, tokens = torch.finfo(c.dtype).eps / 2, ql.shape[1]
    kinds = set()
    for b, n in enumerate(c.lens):
        x = rows[b].double()
        size_x = torch.where(torch.isfinite(x), x, 0.0).abs()
        for t in range(tokens):
            k = max(0, n - (tokens - 1 - t))
            o, s = out[b, t].double(), lse[b, t].double()
            if not k:
                assert (o == 0).all() and (s == -math.inf).all()
                continue
            q = torch.cat([ql[b, t], qr[b, t]], -1).double()
            a = scale * q @ x[:k].t()
            p = torch.softmax(a, -1)
            want = p @ x[:k, :c.latent]
            bad = torch.isnan(want)
            assert torch.equal(torch.isnan(o), bad), "sequence %d token %d: NaN where none belongs, or none where one does" % (b, t)
            kinds |= {"row" if r.all() else "some" if r.any() else "none" for r in bad}
            ds = float((scale * q.abs() @ size_x[:k].t()).max()) * (c.latent + c.rope) * 2.0 ** -24
            pf = torch.where(torch.isnan(p), 0.0, p)
            bound = pf @ size_x[:k, :c.latent] * (e + 4 * ds + 2.0 ** -18) + e * want.abs() + 2.0 ** -25
            assert ((o - want).abs() <= bound)[~bad].all(), (b, t)
            whole = ~torch.isnan(p).any(-1)
            want_lse = torch.logsumexp(a, -1)
            assert ((s - want_lse).abs() <= ds + 2.0 ** -20 + want_lse.abs() * 2.0 ** -22)[whole].all()
            assert not torch.isfinite(s[~whole]).any()
    return kinds


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens,heads", [([65, 130, 64, 2, 1], 4), ([65, 300, 3], 40), ([20000], 30)])
def test_decode_broken_latents(vk, dtype, bad, lens, heads):
    """Broken latents among the drafted rows and before them, in sequences that one CTA has and that all share."""
    g, tokens, scale = gen(len(lens) + heads), 3, 0.07
    c = Cache(vk, lens, 256, 32, 32, layers=2, layer=1, dtype=dtype)
    ql, qr = rnd(g, len(lens), tokens, heads, 256, dtype=dtype, std=0.5), rnd(g, len(lens), tokens, heads, 32, dtype=dtype)
    view = c.pool.latent_view()

    def spoil(b, key, element, value):
        if key >= 0:
            c.rows[b][key, element] = value
            view[1, int(c.tables[b, key // 32]), key % 32, element] = value

    for b, n in enumerate(lens):
        spoil(b, n - 1, 100, bad)  # token 2 sees it
        spoil(b, n - 2, 7, -bad)   # tokens 1 and 2
    out, lse = c.pool.decode(1, ql, qr, c.tables, c.seq_lens, scale, return_lse=True)
    assert c.check() == 0
    kinds = decode_pattern_check(c, c.rows, ql, qr, out, lse, scale)
    assert kinds >= ({"row", "none"} if bad != bad else {"row", "some", "none"})
    again, lse2 = c.pool.decode(1, ql, qr, c.tables, c.seq_lens, scale, return_lse=True)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16)) and torch.equal(lse.view(torch.int32), lse2.view(torch.int32))
    for b, n in enumerate(lens):
        if n > 60:
            spoil(b, 5, 200, bad)  # all tokens see it
    out, lse = c.pool.decode(1, ql, qr, c.tables, c.seq_lens, scale, return_lse=True)
    assert c.check() == 0
    decode_pattern_check(c, c.rows, ql, qr, out, lse, scale)
    # an infinite rotary part: a score of -inf weighs nothing and leaves no element, one of +inf makes the row NaN
    for b, n in enumerate(lens):
        spoil(b, n - 1, 100, 0.5)
        spoil(b, n - 2, 7, 0.5)
        spoil(b, 5 if n > 60 else -1, 200, 0.5)
        spoil(b, n - 1, 256 + 3, bad)
    out, lse = c.pool.decode(1, ql, qr, c.tables, c.seq_lens, scale, return_lse=True)
    assert c.check() == 0
    decode_pattern_check(c, c.rows, ql, qr, out, lse, scale)


def test_decode_rows_that_see_only_infinite_scores(vk):
    """One cached row whose score is -inf: 0/0 by the formula, not the zeros of a row that sees nothing; alone and in
    sequences that several CTAs share."""
    g, scale = gen(77), 0.07
    c = Cache(vk, [1, 0, 1, 4000], 128, 16, 16, layers=1, layer=0)
    ql, qr = rnd(g, 4, 1, 3, 128, std=0.5), rnd(g, 4, 1, 3, 16)
    ql[..., 9] = ql[..., 9].abs() + 0.5
    view = c.pool.latent_view()
    for b, n in enumerate(c.lens):
        c.rows[b][:, 9] = -math.inf
        ids = c.tables[b].repeat_interleave(16)[:n].long()
        view[0, ids, torch.arange(n, device="cuda") % 16, 9] = -math.inf
    out, lse = c.pool.decode(0, ql, qr, c.tables, c.seq_lens, scale, return_lse=True)
    assert c.check() == 0
    for b in (0, 2, 3):
        assert torch.isnan(out[b]).all() and (lse[b] == -math.inf).all()
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


# ------------------------------------------------------------------ groups of sequences


def test_prefill_workspace_bound_and_groups_of_sequences(vk):
    """Bounds so wide that one head of all sequences takes more than the workspace's 1 GiB: sequences go in groups."""
    g = gen(91)
    lens = torch.randint(1, 200, (37,), generator=g, device="cuda").tolist()
    lens[3], lens[20] = 0, 300
    new = [min(n, 1 + 7 * i % 150) for i, n in enumerate(lens)]
    c = Cache(vk, lens, 128, 16, 64, layers=1, layer=0)
    bound = 65536  # 37 * 65536 rows of 512 bytes: 1.16 GiB a head
    c.tables = torch.cat([c.tables, torch.full((37, bound // 64 - c.tables.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    parts = c.pool.prefill_workspace_size(1, 1, 1) - 128 * 512
    for batch, longest, heads in ((37, bound, 3), (37, bound, 1), (32, 131072, 40), (1000, 8192, 5), (65535, 128, 9), (4000, 1 << 20, 2)):
        size = c.pool.prefill_workspace_size(batch, longest, heads)
        assert 0 < size <= max(1 << 30, -(-longest // 128) * 128 * 512) + parts, (batch, longest, heads)
    prefill_check(c, g, new, 3, max_tokens=150, max_seq_len=bound)
    # without bounds: what the tables hold
    prefill_check(c, g, new, 2)


# ------------------------------------------------------------------ offsets of a part of a batch


def test_offsets_of_a_part_of_a_batch(vk):
    """offsets[k:k+n+1] of a larger batch: the rows of the sequences before and behind are ignored, by the append and by
    the prefill, and nothing is recorded."""
    g = gen(95)
    c = Cache(vk, [40, 30, 70], layers=1, layer=0)
    new = [3, 20, 5]
    cu = torch.tensor([0, 7, 10, 30, 35, 36], dtype=torch.int32, device="cuda")  # sequences 1..3 of 5
    start = c.seq_lens - torch.tensor(new, dtype=torch.int32, device="cuda")
    kv = rnd(g, 36, 576)
    before = c.pool.latent_view().clone()
    c.pool.append(0, kv[:, :512], kv[:, 512:], c.tables, start, offsets=cu[1:5])
    assert c.check() == 0
    for b in range(3):
        rows = kv[int(cu[b + 1]):int(cu[b + 2])]
        for i in range(new[b]):
            pos = int(start[b]) + i
            before[0, int(c.tables[b, pos // 16]), pos % 16] = rows[i]
    assert torch.equal(c.pool.latent_view().view(torch.int16), before.view(torch.int16))
    q, w = rnd(g, 36, 2, 192), rnd(g, 512, 512, std=512 ** -0.5)
    out = torch.full((36, 2, 128), 9.0, device="cuda").half()
    c.pool.prefill(0, q, w, c.tables, start, offsets=cu[1:5], max_tokens=20, max_seq_len=70, out=out)
    assert c.check() == 0
    assert (out[:7] == 9).all() and (out[35:] == 9).all()
    want = c.pool.prefill(0, q[7:35].contiguous(), w, c.tables, start, offsets=cu[1:5] - 7, max_tokens=20, max_seq_len=70)
    assert torch.equal(out[7:35], want)


# ------------------------------------------------------------------ host threads


def test_calls_from_host_threads(vk):
    """Four host threads, a stream each, call every entry point of one pool at once."""
    import threading
    g = gen(97)
    c = Cache(vk, [300, 70], 384, 48, 32, layers=5, layer=0)
    view = c.pool.latent_view()
    view[1:] = 0
    ql, qr = rnd(g, 2, 1, 8, 384, std=0.5), rnd(g, 2, 1, 8, 48)
    q, w, kv = rnd(g, 2, 20, 3, 176), rnd(g, 3 * 256, 384, std=384 ** -0.5), rnd(g, 40, 432)
    rope = vk.RotaryEmbedding(48, layout="half")
    want = c.pool.decode(0, ql, qr, c.tables, c.seq_lens, 0.07), c.pool.prefill(0, q, w, c.tables, c.seq_lens - 20)
    torch.cuda.synchronize()
    got, failed = [], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            for _ in range(5):
                c.pool.append(1 + i, kv[:, :384], kv[:, 384:], c.tables, c.seq_lens - 20, rope=rope, stream=s)
                got.append((c.pool.decode(0, ql, qr, c.tables, c.seq_lens, 0.07, stream=s),
                            c.pool.prefill(0, q, w, c.tables, c.seq_lens - 20, stream=s)))
            s.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and c.check() == 0
    assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got)
    for i in range(1, 4):
        assert torch.equal(view[1].view(torch.int16), view[1 + i].view(torch.int16))


# ------------------------------------------------------------------ more heads than a unit's rows


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,tokens", [([30000], 1), ([9000, 20011, 64, 1, 12345], 1), ([4000, 7001], 2)])
def test_decode_128_heads_over_long_contexts(vk, dtype, lens, tokens):
    g = gen(len(lens) + 200)
    c = Cache(vk, lens, page=64, layers=1, layer=0, dtype=dtype)
    n = len(lens)
    ql, qr = rnd(g, n, tokens, 128, 512, dtype=dtype, std=0.5), rnd(g, n, tokens, 128, 64, dtype=dtype)
    out, lse = c.pool.decode(0, ql, qr, c.tables, c.seq_lens, scale=0.07, return_lse=True)
    assert c.check() == 0
    decode_bound_check(c, ql, qr, out, lse, 0.07, tokens)


# ------------------------------------------------------------------ pools, and calls with nothing in them


def test_a_new_pool_is_zero_before_any_stream_uses_it(vk):
    """Memory of the library's own: the zero fill is over when the pool is there, also for a stream that waits for nothing."""
    g = gen(98)
    kv = rnd(g, 64, 576)
    p = torch.zeros(64, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    pages = (12 << 30) // (16 * 576 * 2)
    tables = torch.arange(pages - 64, pages, dtype=torch.int32, device="cuda")[:, None].contiguous()
    ql, qr = rnd(g, 64, 8, 512), rnd(g, 64, 8, 64)
    torch.cuda.synchronize()
    small = vk.LatentKVPool(1, 512, 64, 64)
    small.append(0, kv[:, :512], kv[:, 512:], tables - (pages - 64), p)
    want = small.decode(0, ql, qr, tables - (pages - 64), p + 1, 0.07)
    torch.cuda.synchronize()
    pool = vk.LatentKVPool(1, 512, 64, pages, own_memory=True)
    pool.append(0, kv[:, :512], kv[:, 512:], tables, p, stream=s)
    s.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(pool.decode(0, ql, qr, tables, p + 1, 0.07), want)
    assert pool.check() == 0
    pool.close()


def test_batches_without_tokens(vk):
    """[batch, 0, heads, d]: nothing to do, in every entry point that takes batches."""
    c = Cache(vk, [40, 20])
    empty = lambda heads, d: torch.empty(2, 0, heads, d, device="cuda").half()  # noqa: E731
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert vk.RotaryEmbedding(64).apply(empty(3, 64), none).shape == (2, 0, 3, 64)
    out, lse = c.pool.decode(0, empty(4, 512), empty(4, 64), c.tables, c.seq_lens, 0.1, return_lse=True)
    assert out.shape == (2, 0, 4, 512) and lse.shape == (2, 0, 4)
    assert c.pool.prefill(0, empty(3, 192), rnd(gen(1), 768, 512), c.tables, c.seq_lens).shape == (2, 0, 3, 128)
    assert c.check() == 0


def test_bounds_beyond_the_prefill_are_refused_before_memory_is_taken(vk):
    """Tables wider than the longest sequence that a call takes, without a bound: refused, not an allocation of terabytes."""
    c = Cache(vk, [40], 128, 16, 64)
    q, w = rnd(gen(2), 1, 8, 2, 144), rnd(gen(3), 512, 128)
    wide = torch.full((1, 1 << 22), -1, dtype=torch.int32, device="cuda")
    wide[0, 0] = c.tables[0, 0]
    assert c.pool.prefill_workspace_size(1, (1 << 22) * 64, 2) == 0
    with pytest.raises(vk.VKError, match="max_seq_len"):
        c.pool.prefill(1, q, w, wide, c.seq_lens - 8)
    got = c.pool.prefill(1, q, w, wide, c.seq_lens - 8, max_seq_len=40)
    assert torch.equal(got, c.pool.prefill(1, q, w, c.tables, c.seq_lens - 8, max_seq_len=40)) and c.check() == 0
