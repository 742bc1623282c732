"""GPU: the 8-bit key/value cache - append against a restatement of its rule with the framework's own Quantize / Dequantize
arithmetic (equal bits), attention against a 64-bit softmax over the dequantised cache (tolerances from the roundings that the
kernel makes)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]
TINY = np.float32(2.0 ** -126)


def f32_codes(x, scale):
    """Quantize(x, {scale, 128}): every step rounded to float, halves away from zero."""
    with np.errstate(all="ignore"):
        v = np.float32(128) + (x.astype(np.float32) / np.float32(scale)).astype(np.float32)
    return np.floor(np.clip(v.astype(np.float32), 0, 255).astype(np.float64) + 0.5).astype(np.uint8)


class Model:
    """The cache as numpy arrays, appended to by the rule in include/ltq.h."""

    def __init__(self, cache):
        self.codes = {n: getattr(cache, n).cpu().numpy().copy() for n in "kv"}
        self.scale = {n: getattr(cache, n + "_qparams").cpu().numpy().view(np.float32)[..., 0].copy() for n in "kv"}
        self.bt = cache.block_tokens

    def append(self, new, table, lengths, offsets):
        for b in range(len(lengths)):
            n = int(offsets[b + 1] - offsets[b])
            for p in range(max(0, int(lengths[b]) - n) // self.bt * self.bt, int(lengths[b]), self.bt) if n else ():
                self._block(new, int(table[b][p // self.bt]), p, int(lengths[b]), n, int(offsets[b]))

    def _block(self, new, page, first, length, n, off):
        if not 0 <= page < self.codes["k"].shape[0]:
            return
        start = max(0, length - n)
        used, end = max(0, start - first), min(self.bt, length - first)
        rows = [off + first + i - (length - n) for i in range(used, end)]
        for name in "kv":
            x = np.stack([new[name][r] for r in rows], 1)             # [heads, tokens, D]
            for h in range(x.shape[0]):
                most = np.abs(x[h]).max()
                need = max(np.float32(most / np.float32(127)), TINY)
                old = self.scale[name][page, h] if used else np.float32(0)
                if not np.isfinite(most) or np.isnan(x[h]).any() or np.isnan(old):
                    self.scale[name][page, h] = np.nan
                    self.codes[name][page, h, used:end] = 128
                    continue
                s = max(need, old)
                if used and s > old:
                    held = old * (self.codes[name][page, h, :used].astype(np.float32) - np.float32(128))
                    self.codes[name][page, h, :used] = f32_codes(held, s)
                self.codes[name][page, h, used:end] = f32_codes(x[h], s)
                self.scale[name][page, h] = s

    def equals(self, cache):
        for n in "kv":
            qp = getattr(cache, n + "_qparams").cpu().numpy()
            if not (np.array_equal(getattr(cache, n).cpu().numpy(), self.codes[n]) and
                    np.array_equal(qp.view(np.float32)[..., 0], self.scale[n], equal_nan=True)):
                return False
        return True


def ints(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def batch(torch, seed, spans, bt, spare=2, wide=0):
    """offsets, lengths, block table of sequences with (new, length) tokens; blocks in random order.  `wide`: that many more
    table columns (the launch is sized by the table's width)."""
    g = torch.Generator().manual_seed(seed)
    per = [-(-max(length, 0) // bt) for _, length in spans]
    blocks = sum(per) + spare
    order = torch.randperm(blocks, generator=g).tolist()
    table = [[order.pop() for _ in range(n)] + [-7] * (max(per + [1]) + wide - n) for n in per]   # unused entries are never read
    offsets = [0]
    for n, _ in spans:
        offsets.append(offsets[-1] + n)
    return dict(offsets=offsets, lengths=[length for _, length in spans], table=table, blocks=blocks, max_new=max(n for n, _ in spans),
                tokens=offsets[-1])


def random_cache(torch, ltq, seed, blocks, heads, bt, D):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = ltq.KVCache.empty(blocks, heads, bt, D)
    for n in "kv":
        getattr(cache, n).copy_(torch.randint(0, 256, (blocks, heads, bt, D), generator=g, device="cuda", dtype=torch.uint8))
        qp = getattr(cache, n + "_qparams")
        qp.view(torch.float32)[..., 0] = 0.02 * torch.exp(0.7 * torch.randn(blocks, heads, generator=g, device="cuda"))
        qp[..., 4] = torch.randint(100, 156, (blocks, heads), generator=g, device="cuda", dtype=torch.uint8)
    return cache


# ---- append ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bt,D,heads", [(16, 128, 2), (32, 64, 3), (64, 96, 1), (128, 256, 2), (16, 32, 5), (32, 192, 1)])
def test_append_in_several_calls(cuda, dtype, bt, D, heads):
    """A prompt, then pieces that fill a block part way, to its end and across several blocks; scales grow on the way."""
    import ltq
    torch = cuda
    final = [3 * bt + 5, bt, 1, 2 * bt - 1, 0]
    b = batch(torch, 3, [(0, n) for n in final], bt)
    cache = random_cache(torch, ltq, 1, b["blocks"], heads, bt, D)
    for n in "kv":
        getattr(cache, n + "_qparams")[..., 4] = 128
    model = Model(cache)
    rng = np.random.default_rng(0)
    done = [0] * len(final)
    for piece in (1, 3, bt - 2, 2 * bt + 1, bt + 9, 1, 1):
        take = [min(piece, f - d) for f, d in zip(final, done)]
        done = [d + t for d, t in zip(done, take)]
        offsets = np.concatenate([[0], np.cumsum(take)])
        total = int(offsets[-1])
        if total == 0:
            break
        grow = np.float32(rng.uniform(0.3, 3.0))
        new = {n: torch.from_numpy((grow * rng.standard_normal((total, heads, D))).astype(np.float32)).to(getattr(torch, dtype)) for n in "kv"}
        args = (ints(torch, b["table"]), ints(torch, done), ints(torch, offsets.tolist()), max(take))
        cache.append(new["k"].cuda(), new["v"].cuda(), *args)
        model.append({n: new[n].float().numpy() for n in "kv"}, b["table"], done, offsets)
        assert model.equals(cache)
        cache.append(new["k"].cuda(), new["v"].cuda(), *args)     # the same tokens once more change nothing
        assert model.equals(cache)
    cache.check()
    assert (cache.k_qparams[[p for row in b["table"] for p in row if p >= 0]][..., 4] == 128).all()


def test_append_strided_and_unaligned_sources(cuda):
    import ltq
    torch = cuda
    for extra, shift in ((64, 0), (3, 1), (8, 4)):
        b = batch(torch, 4, [(20, 25), (7, 7)], 16)
        cache = ltq.KVCache.empty(b["blocks"], 2, 16, 64)
        model = Model(cache)
        wide = torch.randn(27, 2 * 128 + extra).half()
        dev = wide.cuda()
        k, v = (dev[:, shift + 128 * i:shift + 128 * (i + 1)].unflatten(1, (2, 64)) for i in range(2))
        cache.append(k, v, ints(torch, b["table"]), ints(torch, b["lengths"]), ints(torch, b["offsets"]), 20)
        model.append({"k": k.float().cpu().numpy(), "v": v.float().cpu().numpy()}, b["table"], b["lengths"], b["offsets"])
        assert model.equals(cache)


def test_append_values_that_are_not_finite_or_vanish(cuda):
    """One block's scale of one head becomes NaN and stays so; zeros and subnormals get the smallest scale."""
    import ltq
    torch = cuda
    b = batch(torch, 5, [(40, 40)], 16)
    cache = ltq.KVCache.empty(b["blocks"], 2, 16, 32)
    model = Model(cache)
    k, v = torch.randn(40, 2, 32), torch.randn(40, 2, 32)
    k[17, 1, 3] = float("inf")
    v[3, 0, 0] = float("nan")
    v[32:] = 0
    k[32:] = 1e-42
    args = (ints(torch, b["table"]), ints(torch, [40]), ints(torch, [0, 40]), 40)
    cache.append(k.cuda(), v.cuda(), *args)
    model.append({"k": k.numpy(), "v": v.numpy()}, b["table"], [40], [0, 40])
    assert model.equals(cache)
    assert torch.isnan(cache.k_qparams.view(torch.float32)[..., 0]).sum() == 1
    more = torch.randn(1, 2, 32)      # behind a finite start in the last block: its scale grows from 2^-126
    cache.append(more.cuda(), more.cuda(), ints(torch, b["table"]), ints(torch, [41]), ints(torch, [0, 1]), 1)
    model.append({"k": more.numpy(), "v": more.numpy()}, b["table"], [41], [0, 1])
    assert model.equals(cache)
    again = torch.randn(12, 2, 32)    # rewriting the tail of the poisoned block leaves it poisoned
    cache.append(again.cuda(), again.cuda(), ints(torch, b["table"]), ints(torch, [32]), ints(torch, [0, 12]), 12)
    model.append({"k": again.numpy(), "v": again.numpy()}, b["table"], [32], [0, 12])
    assert model.equals(cache)


def test_append_padding_and_sequences_out_of_bounds(cuda):
    """Tokens in front of position 0 are not stored; a sequence or block id that contradicts the bounds is left out and
    reported once; the others are stored."""
    import ltq
    torch = cuda
    bt = 16
    cache = ltq.KVCache.empty(8, 1, bt, 32)
    model = Model(cache)
    k = torch.randn(30, 1, 32)
    table = [[0, 1], [2, 3], [4, 99], [5, 6]]
    lengths, offsets = [3, 33, 20, 5], [0, 6, 10, 25, 30]       # six rows for three tokens; 33 > 2 * 16; block 99
    cache.append(k.cuda(), k.cuda(), ints(torch, table), ints(torch, lengths), ints(torch, offsets), 15)
    ok = [0, 2, 3]
    for i in ok:
        model.append({"k": k.numpy(), "v": k.numpy()}, [table[i]], [lengths[i]], offsets[i:i + 2])
    assert model.equals(cache)
    with pytest.raises(ltq.LtqError) as e:
        cache.check()
    assert e.value.status == -1
    cache.check()
    before = {n: getattr(cache, n).clone() for n in "kv"}
    for bad in ([0, 40], [0, -1], [5, 3], [-2, 1]):             # offsets that leave [0, tokens] or fall, more than max_new
        cache.append(k.cuda(), k.cuda(), ints(torch, [[0, 1]]), ints(torch, [20]), ints(torch, bad), 15)
        with pytest.raises(ltq.LtqError):
            cache.check()
    cache.append(k.cuda(), k.cuda(), ints(torch, [[0, 1]]), ints(torch, [-4]), ints(torch, [0, 3]), 15)
    with pytest.raises(ltq.LtqError):
        cache.check()
    assert all(torch.equal(before[n], getattr(cache, n)) for n in "kv")


# ---- attention ------------------------------------------------------------------------------------------------------------

def attention_want(torch, cache, q, b, scale):
    """float64 output and the allowed distance from it, per element."""
    D, bt, heads = cache.head_dim, cache.block_tokens, cache.kv_heads
    group = q.shape[1] // heads
    val = {n: (getattr(cache, n + "_qparams").view(torch.float32)[..., 0].double()[..., None, None] *
               (getattr(cache, n).double() - getattr(cache, n + "_qparams")[..., 4].double()[..., None, None])) for n in "kv"}
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    eps = torch.finfo(q.dtype).eps
    fine = q.dtype == torch.float32
    for i, length in enumerate(b["lengths"]):
        off, n = b["offsets"][i], b["offsets"][i + 1] - b["offsets"][i]
        pages = torch.tensor(b["table"][i][:-(-length // bt)], device="cuda", dtype=torch.long)
        pos = length - n + torch.arange(n, device="cuda")
        live = pos >= 0
        for h in range(heads if bool(live.any()) else 0):
            k, v = (val[x][pages, h].reshape(-1, D)[:length] for x in "kv")
            qq = q[off:off + n, h * group:(h + 1) * group].double()[live]
            seen = (torch.arange(length, device="cuda") <= pos[live][:, None])[:, None]
            s = (qq @ k.t() * scale).masked_fill(~seen, -math.inf)
            rows = slice(off + n - int(live.sum()), off + n)
            want[rows, h * group:(h + 1) * group] = torch.softmax(s, 2) @ v
            # scores: q to 2^-22 of its largest entry (float) or exact, products summed in float by the tensor core
            # (at most 2^-23 per addition), one more rounding each for the two scales and the subtraction of the maximum
            size = (qq.abs() @ k.abs().t()).masked_fill(~seen, 0).amax(2, keepdim=True) + qq.abs().amax(2, keepdim=True) * k.abs().sum(1).amax()
            ds = abs(scale) * size * (2.0 ** -22 + D * 2.0 ** -23 + 4 * 2.0 ** -24)
            # probabilities: 2^-11 (half) or 2^-22 (two halves) relative, the exponential's 2^-22; sums in float.  Subnormal halves
            # are off by 2^-25: in units of v's reference scale, at most twice the largest of the row's, times codes up to twice
            # the largest value's, over a sum of at least 1/2 (the reference maximum is rounded up to an integer): 2^-22 per key
            keys = (pos[live] + 1)[:, None, None]
            dp = 2 * ds + (2.0 ** -21 if fine else 2.0 ** -11) + 2.0 ** -21 + keys * 2.0 ** -23 + keys * 2.0 ** -22
            largest = torch.cummax(v.abs(), 0).values[pos[live]][:, None]
            tol[rows, h * group:(h + 1) * group] = dp * largest + 1e-300
    return want, tol + eps / 2 * (want.abs() + tol)


CASES = [  # spans, block_tokens, head_dim, kv_heads, group
    ([(1, 1)], 16, 128, 1, 1), ([(1, 15), (1, 16), (1, 17)], 16, 64, 2, 4), ([(1, 100), (1, 333), (1, 1)], 32, 128, 2, 8),
    ([(1, 700)], 64, 128, 1, 12), ([(1, 2000), (1, 5)], 128, 96, 1, 7), ([(3, 40), (1, 129), (5, 5)], 16, 32, 2, 3),
    ([(33, 100), (2, 260)], 64, 64, 2, 2), ([(70, 70)], 32, 256, 1, 2), ([(20, 513), (0, 30)], 16, 192, 2, 5), ([(6, 3), (2, 0), (1, 50)], 16, 128, 1, 4),
    ([(129, 300)], 128, 128, 2, 4), ([(100, 100)], 16, 64, 1, 1), ([(40, 513), (64, 64), (3, 700), (130, 90)], 32, 128, 2, 4),
    ([(65, 90 + i) for i in range(40)], 16, 128, 2, 2), ([(40, 70 + 3 * i) for i in range(80)], 32, 256, 1, 2),
    ([(600, 700)], 16, 64, 2, 4), ([(700, 700), (0, 5)], 16, 32, 1, 24), ([(300, 305)], 128, 96, 2, 4),
    ([(128, 128)], 128, 96, 1, 2), ([(50, 900)], 64, 192, 2, 3), ([(300, 333)], 64, 256, 1, 1), ([(65, 1000), (0, 5)], 16, 32, 2, 3),
    ([(1, 4100), (1, 4096), (1, 31)], 64, 128, 2, 16),
    # more groups of rows than the device takes at once: dealt out by what they see, and too many for that
    ([(1 + 37 * i % 200, 60 + 211 * i % 700) for i in range(40)], 32, 64, 2, 4),
    ([(300, 320)] + [(1 + i % 5, 20 + i) for i in range(299)], 16, 32, 1, 4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("wide", [0, 20000])
def test_attention(cuda, dtype, case, wide):
    """Tables as wide as the sequences need (few keys: one launch) and far wider (work divided on the device, parts joined)."""
    import ltq
    torch = cuda
    spans, bt, D, heads, group = CASES[case]
    b = batch(torch, case, spans, bt, wide=wide // bt)
    cache = random_cache(torch, ltq, case, b["blocks"], heads, bt, D)
    q = torch.randn(b["tokens"], heads * group, D, generator=torch.Generator().manual_seed(case)).to(getattr(torch, dtype)).cuda()
    got = cache.attention(q, ints(torch, b["table"]), ints(torch, b["lengths"]), ints(torch, b["offsets"]), b["max_new"])
    cache.check()
    want, tol = attention_want(torch, cache, q, b, D ** -0.5)
    assert got.dtype == q.dtype
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got.double() - want).abs() / tol).max():.3g} of the tolerance"


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_sharp_large_and_small_scores(cuda, dtype):
    """Maxima that keep rising along the keys, scores of thousands, queries far from 1 in size, a zero query, one scale."""
    import ltq
    torch = cuda
    b = batch(torch, 9, [(1, 900), (2, 650)], 16)
    cache = random_cache(torch, ltq, 9, b["blocks"], 2, 16, 64)
    for i, row in enumerate(b["table"]):
        for j, page in enumerate(row):
            if page >= 0:
                cache.k_qparams.view(torch.float32)[page, :, 0] = 0.002 * 1.12 ** j
    q = torch.randn(3, 6, 64)
    q[:, 1] *= 300
    q[:, 2] *= 3e-5
    q[:, 3] = 0
    q[:, 4] *= torch.logspace(-3, 1, 64)
    q = q.to(getattr(torch, dtype)).cuda()
    args = (ints(torch, b["table"]), ints(torch, b["lengths"]), ints(torch, b["offsets"]), 2)
    for scale in (0.125, 3.0, -0.5, 0.0):
        got = cache.attention(q, *args, scale=scale)
        want, tol = attention_want(torch, cache, q, b, float(np.float32(scale)))
        loose = tol > 1   # where scores are so large that their own rounding moves probabilities freely, nothing is said
        assert not ((got.double() - want).abs() > tol)[~loose].any()
        assert torch.isfinite(got).all()
        inside = cache.values()[1].abs().max()
        assert (got.abs() <= inside * (1 + 2 ** -7)).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_prompt_attention_sharp_scores_and_growing_scales(cuda, dtype, head_dim):
    """The same for rows enough to fill the large tiles: the maximum and the largest v scale rise, or fall, from block to block."""
    import ltq
    torch = cuda
    b = batch(torch, 15, [(260, 2300), (150, 900), (300, 300)], 16)
    cache = random_cache(torch, ltq, 15, b["blocks"], 2, 16, head_dim)
    for up_k, up_v in ((1.04, 1.06), (0.97, 0.96), (1.03, 0.97)):
        for row in b["table"]:
            for j, page in enumerate(row):
                if page >= 0:
                    cache.k_qparams.view(torch.float32)[page, :, 0] = 0.002 * up_k ** j
                    cache.v_qparams.view(torch.float32)[page, :, 0] = 0.01 * up_v ** j
        q = torch.randn(b["tokens"], 6, head_dim, generator=torch.Generator().manual_seed(head_dim))
        q[:, 1] *= 30
        q[:, 2] *= 3e-5
        q[::7, 3] = 0
        q = q.to(getattr(torch, dtype)).cuda()
        args = (ints(torch, b["table"]), ints(torch, b["lengths"]), ints(torch, b["offsets"]), b["max_new"])
        for scale in (head_dim ** -0.5, -0.3, 0.0):
            got = cache.attention(q, *args, scale=scale)
            want, tol = attention_want(torch, cache, q, b, float(np.float32(scale)))
            largest = cache.values()[1].abs().max()
            loose = tol > largest   # scores so large that their own rounding moves probabilities freely
            assert not ((got.double() - want).abs() > tol)[~loose].any()
            assert torch.isfinite(got).all() and (got.abs() <= largest * (1 + 2 ** -7)).all()
            assert torch.equal(cache.attention(q, *args, scale=scale), got)


def test_attention_ignores_what_it_may_not_see(cuda):
    """Keys behind the length, other blocks and, for earlier new tokens, later ones: infinities of theirs do not leak in."""
    import ltq
    torch = cuda
    for spans in ([(4, 70)], [(1, 33)], [(40, 100)]):
        b = batch(torch, 11, spans, 16)
        cache = random_cache(torch, ltq, 11, b["blocks"], 2, 16, 128)
        q = torch.randn(b["tokens"], 8, 128).bfloat16().cuda()
        args = (ints(torch, b["table"]), ints(torch, b["lengths"]), ints(torch, b["offsets"]), b["max_new"])
        want = cache.attention(q, *args)
        used = [p for p in b["table"][0] if p >= 0]
        idle = [p for p in range(b["blocks"]) if p not in used]
        cache.k_qparams.view(torch.float32)[idle] = float("nan")
        cache.v_qparams.view(torch.float32)[idle] = float("nan")
        tail = spans[0][1] % 16
        if tail:
            cache.k[used[-1], :, tail:] = 255
            cache.v[used[-1], :, tail:] = 0
        assert torch.equal(cache.attention(q, *args), want)
        # a block that is poisoned: rows that see one of its keys are NaN, the others as before
        cache.v_qparams.view(torch.float32)[used[-1], 1, 0] = float("nan")
        got = cache.attention(q, *args)
        n, length = spans[0]
        first = (length - 1) // 16 * 16
        sees = torch.tensor([length - n + t >= first for t in range(n)], device="cuda")
        assert torch.isnan(got[sees][:, 4:]).all() and torch.equal(got[:, :4], want[:, :4]) and torch.equal(got[~sees], want[~sees])


def test_attention_query_that_is_not_finite(cuda):
    import ltq
    torch = cuda
    b = batch(torch, 12, [(1, 50), (3, 20)], 16)
    cache = random_cache(torch, ltq, 12, b["blocks"], 1, 16, 64)
    for dtype in (torch.float32, torch.float16):
        q = torch.randn(4, 9, 64).to(dtype).cuda()
        args = (ints(torch, b["table"]), ints(torch, b["lengths"]), ints(torch, b["offsets"]), 3)
        want = cache.attention(q, *args)
        q[0, 3, 5], q[2, 8, 0] = float("inf"), float("nan")
        got = cache.attention(q, *args)
        assert torch.isnan(got[0, 3]).all() and torch.isnan(got[2, 8]).all()
        keep = torch.ones(4, 9, dtype=torch.bool, device="cuda")
        keep[0, 3] = keep[2, 8] = False
        assert torch.equal(got[keep], want[keep])


def test_attention_empty_rows_and_bad_arguments(cuda):
    """Rows without keys are zero; a sequence out of bounds leaves its rows alone, a bad block's keys do not exist."""
    import ltq
    torch = cuda
    cache = random_cache(torch, ltq, 13, 6, 1, 16, 32)
    q = torch.randn(12, 2, 32).half().cuda()
    table, lengths, offsets = [[0, 1], [2, 3], [4, 77], [5, 0]], [2, 0, 30, 33], [0, 4, 6, 9, 12]
    out = torch.full_like(q, 5.0)
    cache.attention(q, ints(torch, table), ints(torch, lengths), ints(torch, offsets), 4, out=out)
    with pytest.raises(ltq.LtqError) as e:
        cache.check()
    assert e.value.status == -1
    assert (out[:2] == 0).all() and (out[4:6] == 0).all() and (out[9:] == 5.0).all()
    b = dict(lengths=[16], offsets=[0, 1], table=[[4]])
    for t in range(3):     # positions 27, 28, 29: block 77 leaves the first sixteen keys
        want, tol = attention_want(torch, cache, q[6 + t:7 + t], b, 32 ** -0.5)
        assert ((out[6 + t].double() - want[0]).abs() <= tol[0]).all()
    assert (out[2:4] != 0).any()


def test_attention_strided_queries_own_buffers_and_streams(cuda):
    import ltq
    torch = cuda
    b = batch(torch, 14, [(1, 3000), (1, 2500)], 32)
    cache = random_cache(torch, ltq, 14, b["blocks"], 2, 32, 128)
    wide = torch.randn(2, 8 * 128 + 300).bfloat16().cuda()
    args = (ints(torch, b["table"]), ints(torch, b["lengths"]), ints(torch, b["offsets"]), 1)
    for first in (0, 3, 256):
        q = wide[:, first:first + 8 * 128].unflatten(1, (8, 128))
        want = cache.attention(q.contiguous(), *args)
        assert torch.equal(cache.attention(q, *args), want)
        out = torch.empty_like(want)
        ws = torch.empty(cache.attention_workspace(2, 8, 2, len(b["table"][0]), 1), dtype=torch.uint8, device="cuda").fill_(255)
        assert cache.attention(q, *args, out=out, workspace=ws) is out and torch.equal(out, want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = cache.attention(q, *args)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, want)


def test_prompt_attention_captured_and_on_two_streams(cuda):
    """A captured call follows the lengths and offsets of its replay; two calls at once do not meet."""
    import ltq
    torch = cuda
    big, small = [(260, 2300), (150, 900), (257, 600)], [(40, 1100), (0, 17), (300, 302)]
    b = batch(torch, 17, big, 16)
    cache = random_cache(torch, ltq, 17, b["blocks"], 2, 16, 128)
    q = torch.randn(700, 8, 128, generator=torch.Generator().manual_seed(17)).bfloat16().cuda()
    table = ints(torch, b["table"])
    shapes = []
    for spans in (big, small):
        offsets = [0]
        for n, _ in spans:
            offsets.append(offsets[-1] + n)
        shapes.append((ints(torch, [length for _, length in spans]), ints(torch, offsets)))
    want = [cache.attention(q, table, *shape, 300) for shape in shapes]
    lengths, offsets = (t.clone() for t in shapes[0])
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attention(q, table, lengths, offsets, 300, out=out)
    for k in (0, 1, 0):
        lengths.copy_(shapes[k][0])
        offsets.copy_(shapes[k][1])
        rows = int(shapes[k][1][-1])
        graph.replay()
        assert torch.equal(out[:rows], want[k][:rows])
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for k, stream in enumerate(streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got[k].append(cache.attention(q, table, *shapes[k], 300))
    for stream in streams:
        torch.cuda.current_stream().wait_stream(stream)
    for k in range(2):
        rows = int(shapes[k][1][-1])
        assert all(torch.equal(o[:rows], want[k][:rows]) for o in got[k])
    cache.check()


@pytest.mark.parametrize("spans,heads,group,head_dim", [([(742, 1364), (300, 900)], 4, 1, 64), ([(1, 2293), (1, 73)], 8, 8, 96), ([(1, 3000)] * 9, 1, 7, 256),
                                                        ([(25, 2123)], 2, 12, 128)])
def test_attention_of_float_queries_is_float(cuda, spans, heads, group, head_dim):
    """Error of the whole result, in the 2-norm.  Per probability: 2^-22 each for its two halves and its exponential; its score, of a few
    units, some 2^-24 of itself from each sum of 16 products and of those sums: below 2^-20 together, and independent from key
    to key, which the norm of a sum of them does not enlarge."""
    import ltq
    torch = cuda
    b = batch(torch, 18, spans, 32)
    cache = random_cache(torch, ltq, 18, b["blocks"], heads, 32, head_dim)
    q = torch.randn(b["tokens"], heads * group, head_dim, generator=torch.Generator().manual_seed(18)).cuda()
    scale = 1.0 / float(cache.values()[0].std() * head_dim ** 0.5)
    got = cache.attention(q, ints(torch, b["table"]), ints(torch, b["lengths"]), ints(torch, b["offsets"]), b["max_new"], scale=scale)
    want, _ = attention_want(torch, cache, q, b, float(np.float32(scale)))
    assert (got.double() - want).norm() < 2.0 ** -20 * want.norm()


def test_attention_workspace(cuda):
    """None is needed for a short call, and none may be too small for a long one."""
    import ltq
    torch = cuda
    b = batch(torch, 16, [(1, 40)], 16)
    cache = random_cache(torch, ltq, 16, b["blocks"], 1, 16, 64)
    q = torch.randn(1, 4, 64).half().cuda()
    for width in (len(b["table"][0]), 3000):
        table = ints(torch, [b["table"][0] + [-1] * (width - len(b["table"][0]))])
        args = (q, table, ints(torch, b["lengths"]), ints(torch, b["offsets"]), 1)
        need = cache.attention_workspace(1, 4, 1, width, 1)
        want = cache.attention(*args)
        assert (need == 0) == (width < 3000)
        assert torch.equal(cache.attention(*args, workspace=torch.empty(need, dtype=torch.uint8, device="cuda")), want)
        if need:
            with pytest.raises(ltq.LtqError) as e:
                cache.attention(*args, workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
            assert e.value.status == -1
            with pytest.raises(ltq.LtqError):
                cache.attention(*args, workspace=torch.empty(0, dtype=torch.uint8, device="cuda"))


def test_long_cache_offsets_beyond_32_bits(cuda):
    """Block ids whose byte offsets pass 2^32: 140 000 blocks of 16 x 8 heads x 256."""
    import ltq
    torch = cuda
    blocks, heads, bt, D = 140_000, 8, 16, 256
    k = torch.empty((blocks, heads, bt, D), dtype=torch.uint8, device="cuda").fill_(128)
    v = torch.empty_like(k).fill_(128)
    qp = [torch.zeros((blocks, heads, 8), dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache = ltq.KVCache(k, qp[0], v, qp[1])
    pages = [139_999, 3, 135_000]
    small = ltq.KVCache.empty(3, heads, bt, D)
    new = [torch.randn(40, heads, D).half().cuda() for _ in range(2)]
    q = torch.randn(40, heads, D).half().cuda()
    outs = []
    for c, ids in ((cache, pages), (small, [0, 1, 2])):
        args = (ints(torch, [ids]), ints(torch, [40]), ints(torch, [0, 40]), 40)
        c.append(*new, *args)
        outs.append(c.attention(q, *args))
        c.check()
    assert torch.equal(*outs)
    assert torch.equal(cache.k[pages], small.k) and torch.equal(cache.v_qparams[pages], small.v_qparams)
    assert int((cache.k != 128).sum()) == int((small.k != 128).sum())


# ---- together -------------------------------------------------------------------------------------------------------------

def test_decode_steps_of_an_attention_layer_eager_and_captured(cuda):
    """x -> fused q/k/v projection -> append -> attention -> output projection, a prompt and then single tokens; the captured step
    is replayed with lengths and tokens that move on, and agrees with the eager one bit for bit."""
    import ltq
    torch = cuda
    heads, kv, D, width, bt = 8, 2, 64, 256, 16
    g = torch.Generator().manual_seed(0)
    qkv = ltq.FullyConnected_t.from_float(torch.randn((heads + 2 * kv) * D, width, generator=g).mul_(0.06).cuda(), torch.randn((heads + 2 * kv) * D, generator=g).cuda())
    proj = ltq.FullyConnected_t.from_float(torch.randn(width, heads * D, generator=g).mul_(0.05).cuda())
    caches = [ltq.KVCache.empty(12, kv, bt, D) for _ in range(2)]
    table = ints(torch, [[7, 2, 9, 4], [1, 11, 0, 3]])

    def layer(cache, x, lengths, offsets, max_new):
        y = qkv.forward(x).unflatten(1, (heads + 2 * kv, D))
        cache.append(y[:, heads:heads + kv], y[:, heads + kv:], table, lengths, offsets, max_new)
        return proj.forward(cache.attention(y[:, :heads], table, lengths, offsets, max_new).flatten(1)), y

    prompt = torch.randn(30, width, generator=g).bfloat16().cuda()
    for c in caches:
        out, y = layer(c, prompt, ints(torch, [20, 10]), ints(torch, [0, 20, 30]), 20)
    # every stage against its own reference on the stage's actual input
    b = dict(lengths=[20, 10], offsets=[0, 20, 30], table=table.tolist())
    att = caches[0].attention(y[:, :heads], table, ints(torch, [20, 10]), ints(torch, [0, 20, 30]), 20)
    want, tol = attention_want(torch, caches[0], y[:, :heads], b, D ** -0.5)
    assert ((att.double() - want).abs() <= tol).all()
    model = Model(ltq.KVCache.empty(12, kv, bt, D))
    yn = y.float().cpu().numpy()
    model.append({"k": yn[:, heads:heads + kv], "v": yn[:, heads + kv:]}, b["table"], b["lengths"], b["offsets"])
    assert model.equals(caches[0])

    x, lengths, offsets = torch.zeros(2, width, dtype=torch.bfloat16, device="cuda"), ints(torch, [20, 10]), ints(torch, [0, 1, 2])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    lengths += 1
    with torch.cuda.graph(graph):
        captured, _ = layer(caches[1], x, lengths, offsets, 1)
    for step in range(40):
        if int(lengths.max()) > 64:
            break
        new = torch.randn(2, width, generator=g).bfloat16().cuda()
        eager, _ = layer(caches[0], new, lengths.clone(), offsets, 1)
        x.copy_(new)
        graph.replay()
        assert torch.equal(captured, eager)
        lengths += 1
    for n in ("k", "v", "k_qparams", "v_qparams"):
        assert torch.equal(getattr(caches[0], n), getattr(caches[1], n))
    caches[0].check()


def test_refusals(cuda):
    import ltq
    torch = cuda
    cache = ltq.KVCache.empty(4, 2, 16, 64)
    table, lengths, offsets = ints(torch, [[0, 1]]), ints(torch, [5]), ints(torch, [0, 2])
    k, q = torch.randn(2, 2, 64).cuda(), torch.randn(2, 4, 64).cuda()
    args = (table, lengths, offsets, 2)
    for bad in (lambda: cache.append(k[:, :1], k[:, :1], *args), lambda: cache.append(k.cpu(), k.cpu(), *args), lambda: cache.append(k, k.half(), *args),
                lambda: cache.append(k.double(), k.double(), *args), lambda: cache.append(k.transpose(1, 2).contiguous().transpose(1, 2), k, *args),
                lambda: cache.append(k, k, table.long(), lengths, offsets, 2), lambda: cache.append(k, k, table, lengths, offsets[:1], 2),
                lambda: cache.attention(q[..., :32], *args), lambda: cache.attention(q.double(), *args),
                lambda: cache.attention(q, *args, out=torch.empty(2, 4, 64, dtype=torch.half, device="cuda")),
                lambda: cache.attention(q, table.cpu(), lengths, offsets, 2),
                lambda: ltq.KVCache(cache.k, cache.k_qparams[:1], cache.v, cache.v_qparams), lambda: ltq.KVCache(cache.k.float(), cache.k_qparams, cache.v, cache.v_qparams)):
        with pytest.raises(ValueError):
            bad()
    for status, bad in ((-1, lambda: cache.attention(q[:, :3].contiguous(), *args)), (-1, lambda: cache.append(k, k, table, lengths, offsets, 3)),
                        (-1, lambda: cache.attention(q, *args, scale=math.inf)),
                        (-2, lambda: ltq.KVCache.empty(2, 2, 24, 64).append(k, k, *args)),
                        (-2, lambda: ltq.KVCache.empty(2, 2, 16, 80).attention(torch.randn(2, 2, 80).cuda(), *args))):
        with pytest.raises(ltq.LtqError) as e:
            bad()
        assert e.value.status == status
    cache.append(k[:0], k[:0], table, lengths, ints(torch, [0, 0]), 0)
    assert cache.attention(q[:0], table, lengths, ints(torch, [0, 0]), 0).shape == (0, 4, 64)
