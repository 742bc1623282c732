"""GPU: the edges of cache attention in each of its forms, the one that ran named: what a row may not see, queries and scales that are not finite,
sequences and blocks out of bounds, rows off 16-byte boundaries, rows that belong to no sequence.  (Each form has code of its
own for them.)"""
import pytest

from test_gpu_cache import attention_want, batch, ints, random_cache

pytestmark = pytest.mark.gpu

HALVES = ["float16", "bfloat16"]
# form: kernel, [(new, length)], block_tokens, head_dim, kv_heads, group, table columns beyond the longest sequence
FORMS = {"clusters": ("cache_attention_cluster_kernel", [(4, 70), (3, 40), (1, 100)], 16, 128, 2, 4, 0),
         "device": ("cache_attention_kernel", [(4, 70), (3, 40), (1, 900)], 16, 128, 2, 4, 1200),
         "device, 256": ("cache_attention_kernel", [(6, 170), (2, 33)], 32, 256, 1, 3, 700),
         "large, shared": ("cache_attention_tc_kernel", [(300, 2300), (45, 170), (7, 33)], 16, 128, 2, 4, 0),
         "large": ("cache_attention_tc_kernel", [(700, 900), (130, 170), (7, 33)], 64, 128, 8, 4, 0),
         "large, 64": ("cache_attention_tc_kernel", [(600, 700), (200, 450)], 32, 64, 4, 4, 0),
         "large, 256": ("cache_attention_tc_kernel", [(300, 333), (64, 500)], 128, 256, 8, 2, 0),
         "large, 192, shared": ("cache_attention_tc_kernel", [(300, 1500), (20, 64)], 16, 192, 1, 4, 0)}
LARGE = [f for f in FORMS if f.startswith("large")]
SHARED = {"large, shared": True, "large": False, "large, 64": False, "large, 256": False, "large, 192, shared": True}


def case(torch, ltq, form, dtype, spare=3):
    kernel, spans, bt, D, heads, group, wide = FORMS[form]
    b = batch(torch, len(form), spans, bt, spare=spare, wide=wide)
    cache = random_cache(torch, ltq, len(form), b["blocks"], heads, bt, D)
    q = torch.randn(b["tokens"], heads * group, D, generator=torch.Generator().manual_seed(3)).to(getattr(torch, dtype)).cuda()
    args = [ints(torch, b["table"]), ints(torch, b["lengths"]), ints(torch, b["offsets"]), b["max_new"]]
    return cache, q, b, args


def ran(form):
    import ltq
    name = ltq.last_kernel()
    assert name.startswith(FORMS[form][0] + "<"), name
    if form in SHARED:
        assert ("keys in 1)" not in name) == SHARED[form], name


def same(form, got, want):
    """Rows of sequences that another sequence's length has nothing to do with: the same bits.  Only the form that divides the keys of the
    whole batch evenly over the device puts its cuts elsewhere then; its two results are roundings of one sum, each within
    2^-11 (probabilities) + half a step of the type of it in the norm, so within twice that of one another."""
    import torch
    if not form.startswith("device"):
        return torch.equal(got, want)
    bound = 2.0 ** -11 + torch.finfo(want.dtype).eps / 2
    return bool((got.double() - want.double()).norm() <= 2 * bound * want.double().norm())


def positions(torch, b):
    """sequence and position of every row."""
    seq, pos = [], []
    for i, length in enumerate(b["lengths"]):
        n = b["offsets"][i + 1] - b["offsets"][i]
        seq += [i] * n
        pos += range(length - n, length)
    return torch.tensor(seq, device="cuda"), torch.tensor(pos, device="cuda")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("form", FORMS)
def test_against_64_bits(cuda, form, dtype):
    import ltq
    cache, q, b, args = case(cuda, ltq, form, dtype)
    got = cache.attention(q, *args)
    ran(form)
    cache.check()
    want, tol = attention_want(cuda, cache, q, b, q.shape[2] ** -0.5)
    assert not ((got.double() - want).abs() > tol).any()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("which", "kv")
def test_a_scale_of_nan_reaches_the_rows_that_see_its_block(cuda, form, dtype, which):
    """... of its head, and no other row; blocks in no table and codes behind the length reach none."""
    import ltq
    torch = cuda
    cache, q, b, args = case(torch, ltq, form, dtype)
    heads, group, bt = cache.kv_heads, q.shape[1] // cache.kv_heads, cache.block_tokens
    want = cache.attention(q, *args)
    ran(form)
    used = {p for i, row in enumerate(b["table"]) for p in row[:-(-b["lengths"][i] // bt)]}
    idle = [p for p in range(b["blocks"]) if p not in used]
    for n in "kv":
        getattr(cache, n + "_qparams").view(torch.float32)[idle] = float("nan")
    tail = b["lengths"][0] % bt
    if tail:
        last = b["table"][0][b["lengths"][0] // bt]
        cache.k[last, :, tail:] = 255
        cache.v[last, :, tail:] = 0
    assert torch.equal(cache.attention(q, *args), want)
    seq, pos = positions(torch, b)
    # of the first sequence the block that holds the middle of its new tokens, of one head
    middle = b["lengths"][0] - (b["offsets"][1] + 1) // 2
    block = middle // bt
    getattr(cache, which + "_qparams").view(torch.float32)[b["table"][0][block], heads - 1, 0] = float("nan")
    got = cache.attention(q, *args)
    ran(form)
    sees = (seq == 0) & (pos >= block * bt)
    assert sees.any() and torch.isnan(got[sees][:, (heads - 1) * group:]).all()
    assert torch.equal(got[~sees], want[~sees]) and torch.equal(got[:, :(heads - 1) * group], want[:, :(heads - 1) * group])
    cache.check()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("form", FORMS)
def test_queries_that_are_not_finite(cuda, form, dtype):
    import ltq
    torch = cuda
    cache, q, b, args = case(torch, ltq, form, dtype)
    want = cache.attention(q, *args)
    rows = [(0, 0, float("inf")), (b["tokens"] - 1, q.shape[1] - 1, float("nan")), (b["offsets"][1] - 1, 1, float("-inf"))]
    keep = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    for i, (t, h, x) in enumerate(rows):
        q[t, h, 5 * i] = x
        keep[t, h] = False
    got = cache.attention(q, *args)
    ran(form)
    assert torch.isnan(got[~keep]).all() and torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("form", FORMS)
def test_blocks_and_sequences_out_of_bounds(cuda, form, dtype):
    """Keys of a block id out of range do not exist; a sequence that contradicts its bounds is left out, its rows as they were;
    either is reported once, the other sequences are not touched."""
    import ltq
    torch = cuda
    cache, q, b, args = case(torch, ltq, form, dtype)
    bt, D = cache.block_tokens, q.shape[2]
    want = cache.attention(q, *args)
    cache.check()
    first = slice(b["offsets"][0], b["offsets"][1])
    for bad in (b["blocks"], -1, 2 ** 31 - 1):
        table = [list(r) for r in b["table"]]
        table[0][1] = bad
        got = cache.attention(q, ints(torch, table), *args[1:])
        ran(form)
        with pytest.raises(ltq.LtqError, match="block id") as e:
            cache.check()
        assert e.value.status == -1
        cache.check()
        assert torch.equal(got[first.stop:], want[first.stop:])
        # the same keys hidden by scores of their own: a block whose k is far below the others for every row does as well as none
        kept = [p for i, p in enumerate(table[0][:-(-b["lengths"][0] // bt)]) if i != 1]
        val = {n: getattr(cache, n + "_qparams").view(torch.float32)[..., 0].double()[..., None, None] *
               (getattr(cache, n).double() - getattr(cache, n + "_qparams")[..., 4].double()[..., None, None]) for n in "kv"}
        group = q.shape[1] // cache.kv_heads
        pos = b["lengths"][0] - b["offsets"][1] + torch.arange(b["offsets"][1], device="cuda")
        at = torch.cat([torch.arange(bt), torch.arange(2 * bt, (len(kept) + 1) * bt)]).cuda()   # positions of the kept keys
        for h in range(cache.kv_heads):
            k, v = (val[n][kept, h].reshape(-1, D) for n in "kv")
            s = torch.einsum("tgd,kd->tgk", q[first, h * group:(h + 1) * group].double(), k) * D ** -0.5
            s = s.masked_fill((at[None] > pos[:, None])[:, None], float("-inf"))
            o = torch.einsum("tgk,kd->tgd", torch.softmax(s, 2), v)
            diff = got[first, h * group:(h + 1) * group].double() - o
            assert diff.norm() < 2.0 ** (-10 if dtype == "float16" else -7) * o.norm()
    for lengths, offsets in ((None, [b["offsets"][0], b["tokens"] + 1]), ([10 ** 9], None), ([-1], None), (None, [-1, 3])):
        l, o = list(b["lengths"]), list(b["offsets"])
        if lengths:
            l[-1] = lengths[0]
        if offsets:
            o[-1] = offsets[1] if offsets[1] > 3 else -5
        out = torch.full_like(q, 7.0)
        cache.attention(q, args[0], ints(torch, l), ints(torch, o), args[3], out=out)
        ran(form)
        with pytest.raises(ltq.LtqError, match="sequence"):
            cache.check()
        start = b["offsets"][-2]
        assert (out[start:] == 7.0).all() and same(form, out[:start], want[:start])
    cache.check()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("form", FORMS)
def test_rows_off_16_byte_boundaries(cuda, form, dtype):
    """q read and out written at any element offset, token strides of q that are no multiple of eight; nothing beside them is
    written."""
    import ltq
    torch = cuda
    cache, q, b, args = case(torch, ltq, form, dtype)
    want = cache.attention(q, *args)
    row = q.shape[1] * q.shape[2]
    for shift, extra in ((1, 3), (2, 8), (4, 4), (0, 1)):
        wide = torch.zeros(b["tokens"], row + shift + extra, dtype=q.dtype, device="cuda")
        view = wide[:, shift:shift + row]
        view.copy_(q.flatten(1))
        flat = torch.full((b["tokens"] * row + 2 * shift + 8,), 9.0, dtype=q.dtype, device="cuda")
        out = flat[shift:shift + b["tokens"] * row].view(q.shape)
        assert cache.attention(view.unflatten(1, q.shape[1:]), *args, out=out) is out
        ran(form)
        assert torch.equal(out, want)
        assert (flat[:shift] == 9.0).all() and (flat[shift + b["tokens"] * row:] == 9.0).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("form", FORMS)
def test_rows_of_no_sequence_and_rows_without_keys(cuda, form, dtype):
    """Rows behind the last sequence are left as they were; tokens in front of position 0 get zeros; a sequence without tokens of
    this call has no rows."""
    import ltq
    torch = cuda
    cache, q, b, args = case(torch, ltq, form, dtype)
    more = torch.cat([q, q[:5]])
    out = torch.full_like(more, 3.0)
    cache.attention(more, *args, out=out)
    ran(form)
    want = cache.attention(q, *args)
    assert torch.equal(out[:b["tokens"]], want) and (out[b["tokens"]:] == 3.0).all()
    lengths = list(b["lengths"])
    n = b["offsets"][1]
    lengths[0] = n - 3          # three tokens of padding in front
    got = cache.attention(q, args[0], ints(torch, lengths), *args[2:])
    assert (got[:3] == 0).all() and (got[3:n] != 0).any(2).all() and same(form, got[n:], want[n:])
    lengths[0] = 0
    got = cache.attention(q, args[0], ints(torch, lengths), *args[2:])
    assert (got[:n] == 0).all() and same(form, got[n:], want[n:])
    offsets = list(b["offsets"])
    offsets[-1] = offsets[-2]   # the last sequence has no tokens now
    out.fill_(3.0)
    cache.attention(more, args[0], args[1], ints(torch, offsets), args[3], out=out)
    assert same(form, out[:offsets[-1]], want[:offsets[-1]]) and (out[offsets[-1]:] == 3.0).all()
    cache.check()


@pytest.mark.parametrize("form", FORMS)
def test_the_same_bits_at_every_call(cuda, form):
    """... also beside calls on another stream."""
    import ltq
    torch = cuda
    cache, q, b, args = case(torch, ltq, form, "bfloat16")
    want = cache.attention(q, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(20):
        got.append(cache.attention(q, *args))
        with torch.cuda.stream(side):
            got.append(cache.attention(q, *args))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
