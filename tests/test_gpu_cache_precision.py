"""GPU: how exact cache attention is where the blocks' scales differ much, against a 64-bit softmax, in the 2-norm over all outputs.

Bounds.  A probability is rounded to a half (half and bfloat16 queries: off by 2^-11 of itself at most) or to two of them (float queries:
2^-22).  Values are random and of random sign, so a relative error of at most e in every term of a sum, independent from term to
term, is at most e in the norm of the sums.  The output's own rounding adds half a step of its type.  Scores, exponentials and
sums of float queries stay below 2^-20 together (see test_attention_of_float_queries_is_float)."""
import math

import numpy as np
import pytest

from test_gpu_cache import ints

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]
BOUND = {"float32": 2.0 ** -20, "float16": 2.0 ** -11 + 2.0 ** -11, "bfloat16": 2.0 ** -11 + 2.0 ** -8}

# new tokens, keys, block_tokens, head_dim, kv_heads, group, table columns beyond the sequence's
FORMS = {"one launch": (1, 1024, 16, 128, 2, 4, 0), "one launch, 16 rows": (5, 2048, 64, 64, 2, 4, 0), "over the device": (1, 1024, 16, 128, 2, 4, 4000),
         "over the device, 256": (3, 2048, 32, 256, 1, 4, 3000), "one warp per item": (1, 1024, 16, 96, 400, 1, 0),
         "large tiles, keys shared": (300, 2048, 16, 128, 2, 4, 0), "large tiles": (1200, 2048, 64, 128, 8, 4, 0),
         "large tiles, 256": (300, 2048, 128, 256, 8, 4, 0), "large tiles, 32": (700, 1500, 16, 32, 4, 4, 0)}


class Case:
    """One sequence over blocks in order; ordinary blocks of scale 0.02, queries with a common direction so that a block's keys can
    be moved up or down together."""

    def __init__(self, torch, ltq, form, dtype, zero=128):
        self.torch, (self.new, keys, bt, D, heads, group, wide) = torch, FORMS[form]
        g = torch.Generator(device="cuda").manual_seed(len(form) + D)
        n = -(-keys // bt)
        self.keys = keys
        self.cache = c = ltq.KVCache.empty(n, heads, bt, D)
        for x in "kv":
            getattr(c, x).copy_((zero + 36 * torch.randn(n, heads, bt, D, generator=g, device="cuda")).round_().clamp_(1, 255).to(torch.uint8))
            qp = getattr(c, x + "_qparams")
            qp.view(torch.float32)[..., 0] = 0.02
            qp[..., 4] = zero
        self.zero, self.blocks = zero, n
        self.q = (0.5 * torch.randn(self.new, heads * group, D, generator=g, device="cuda") + 0.6).to(getattr(torch, dtype))
        self.scale = 3.0 / math.sqrt(D)
        self.args = (ints(torch, [list(range(n)) + [0] * (wide // bt)]), ints(torch, [keys]), ints(torch, [0, self.new]), self.new)

    def shift(self, block, by):
        """Every score of the block becomes about by * 0.02 * 0.6 * D * scale."""
        self.cache.k[block] = self.zero + by

    def scores(self, block, by, v_scale):
        self.shift(block, by)
        self.cache.v_qparams.view(self.torch.float32)[block, :, 0] = v_scale

    def error(self):
        torch, c, D = self.torch, self.cache, self.cache.head_dim
        got = c.attention(self.q, *self.args, scale=self.scale)
        c.check()
        group = self.q.shape[1] // c.kv_heads
        want = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        val = {n: getattr(c, n + "_qparams").view(torch.float32)[..., 0].double()[..., None, None] *
               (getattr(c, n).double() - getattr(c, n + "_qparams")[..., 4].double()[..., None, None]) for n in "kv"}
        pos = self.keys - self.new + torch.arange(self.new, device="cuda")
        hidden = torch.arange(self.keys, device="cuda")[None] > pos[:, None]
        for h in range(c.kv_heads):
            k, v = (val[n][:, h].reshape(-1, D)[:self.keys] for n in "kv")
            s = torch.einsum("tgd,kd->tgk", self.q[:, h * group:(h + 1) * group].double(), k) * float(np.float32(self.scale))
            want[:, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", torch.softmax(s.masked_fill(hidden[:, None], -math.inf), 2), v)
        assert torch.isfinite(got).all()
        return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS)
def test_a_loud_block_of_v_that_has_no_weight(cuda, form, dtype):
    """Its scores lie 30 and more below the others' (natural logarithm): whatever its scale is, the outputs are those of the others."""
    import ltq
    for louder in (1, 10, 20, 30):
        for where in (0, 1 / 3, 0.6):
            c = Case(cuda, ltq, form, dtype)
            c.scores(int(where * c.blocks), -100, 0.02 * 2.0 ** louder)
            assert c.error() < BOUND[dtype], (louder, where)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS)
def test_scales_of_v_that_grow_and_shrink_along_the_keys(cuda, form, dtype):
    """From block to block by 2^0.5 up to 2^20 and back down, scores against them: the loudest blocks get the least weight."""
    import ltq
    c = Case(cuda, ltq, form, dtype)
    steps = 20.0 * (1 - (2 * cuda.arange(c.blocks, device="cuda") / (c.blocks - 1) - 1).abs())
    c.cache.v_qparams.view(cuda.float32)[..., 0] = (0.02 * 2.0 ** steps)[:, None]
    c.cache.k[:] = (c.cache.k.float() - 4 * steps[:, None, None, None]).round().clamp(0, 255).to(cuda.uint8)
    assert c.error() < BOUND[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("louder", [0, 30])
def test_a_block_of_zeros_that_takes_the_weight(cuda, form, dtype, louder):
    """Values of zero (the smallest scale there is, 2^-126) at the first or a later block, with most of the probability: what is left
    for the others comes out exactly, a loud block without weight beside them or not."""
    import ltq
    for where in (0, 0.5):
        c = Case(cuda, ltq, form, dtype)
        block = int(where * c.blocks)
        c.scores(block, 12, 2.0 ** -126)
        c.cache.v[block] = 128
        if louder:
            c.scores((block + c.blocks // 4) % c.blocks, -100, 0.02 * 2.0 ** louder)
        assert c.error() < BOUND[dtype], where


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [2.0 ** -90, 2.0 ** 90])
def test_values_of_any_size(cuda, form, dtype, size):
    """All of V in another unit: the same outputs in that unit, also beside blocks of the usual one that have no weight."""
    import ltq
    for mixed in (False, True):
        c = Case(cuda, ltq, form, dtype)
        c.cache.v_qparams.view(cuda.float32)[..., 0] = 0.02 * size
        if mixed and size < 1:
            c.scores(c.blocks // 3, -100, 2.0 ** -64)
        if mixed and size > 1:
            c.scores(c.blocks // 3, -100, 0.02)
        assert c.error() < BOUND[dtype], mixed


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("form", FORMS)
def test_one_row_of_a_tile_does_not_take_bits_from_another(cuda, form, dtype):
    """The last block is loud and only the last new tokens see it, with weight: the tokens before it are as exact as without it."""
    import ltq
    c = Case(cuda, ltq, form, dtype)
    if c.new < 2:
        return
    plain = c.cache.attention(c.q, *c.args, scale=c.scale)
    c.cache.v_qparams.view(cuda.float32)[c.blocks - 1, :, 0] = 0.02 * 2.0 ** 12
    assert c.error() < BOUND[dtype]
    got = c.cache.attention(c.q, *c.args, scale=c.scale)
    before = c.new - (c.keys - (c.blocks - 1) * c.cache.block_tokens)
    if before > 0:
        diff = (got[:before].double() - plain[:before].double()).norm() / plain[:before].double().norm()
        assert diff < 2 * BOUND[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS)
def test_blocks_that_were_never_written_are_zeros(cuda, form, dtype):
    """Parameters as KVCache.empty makes them, scale 0: scores and values of zero, whatever the codes are."""
    import ltq
    c = Case(cuda, ltq, form, dtype)
    for block in (1, c.blocks // 2):
        for n in "kv":
            getattr(c.cache, n + "_qparams")[block] = 0
            getattr(c.cache, n)[block] = 200
    assert c.error() < BOUND[dtype]
    for n in "kv":
        getattr(c.cache, n + "_qparams")[:] = 0
    assert (c.cache.attention(c.q, *c.args, scale=c.scale) == 0).all()


# ---- long runs -------------------------------------------------------------------------------------------------------------
# A table may name a block again and again: keys of a few blocks, each with its multiplicity, make long sequences whose 64-bit softmax
# is as quick as that of the few.

LONG = {"decode": (64, 1, 32768, 128, 8, 8), "decode, more sequences": (256, 1, 32768, 128, 8, 8), "decode, 16 heads": (64, 1, 32768, 128, 8, 16),
        "decode, 64": (256, 1, 32768, 64, 8, 4), "decode, 256": (64, 1, 32768, 256, 4, 8), "drafts": (48, 4, 32768, 128, 8, 4),
        "prompt": (2, 300, 131072, 128, 8, 4), "prompt, 256": (2, 300, 65536, 256, 8, 4), "prompt, 64": (2, 600, 65536, 64, 8, 4)}


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("form", LONG)
def test_long_runs_of_keys_do_not_drift(cuda, form, dtype):
    """Nearly flat scores, hundreds to thousands of steps per accumulator: sums that lose a little towards zero at each would show."""
    import ltq
    torch = cuda
    seqs, new, keys, D, heads, group = LONG[form]
    bt, few = 64, 8
    tail = -(-new // bt)
    times = (keys // bt - tail) // few
    g = torch.Generator(device="cuda").manual_seed(7)
    cache = ltq.KVCache.empty(few + tail, heads, bt, D)
    for n in "kv":
        getattr(cache, n).copy_((128 + 36 * torch.randn(few + tail, heads, bt, D, generator=g, device="cuda")).round_().clamp_(0, 255).to(torch.uint8))
        qp = getattr(cache, n + "_qparams")
        qp.view(torch.float32)[..., 0] = 0.02
        qp[..., 4] = 128
    row = list(range(few)) * times + list(range(few, few + tail))
    length, scale = len(row) * bt, float(np.float32(D ** -0.5))
    q = (0.02 * torch.randn(seqs * new, heads * group, D, generator=g, device="cuda")).to(getattr(torch, dtype))
    got = cache.attention(q, ints(torch, [row] * seqs), ints(torch, [length] * seqs), ints(torch, [new * i for i in range(seqs + 1)]), new, scale=scale)
    cache.check()
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    k, v = (0.02 * (getattr(cache, n).double() - 128.0) * (float(np.float32(0.02)) / 0.02) for n in "kv")
    behind = torch.arange((few + tail) * bt, device="cuda") - few * bt          # place of a key behind the repeated ones
    seen = behind[None] <= (tail * bt - new + torch.arange(new, device="cuda"))[:, None]
    often = torch.where(behind < 0, math.log(times), 0.0)
    for h in range(heads):
        kk, vv = k[:, h].reshape(-1, D), v[:, h].reshape(-1, D)
        s = torch.einsum("tgd,kd->tgk", q[:, h * group:(h + 1) * group].double(), kk) * scale + often
        s = s.view(seqs, new, group, -1).masked_fill(~seen[None, :, None], -math.inf)
        want[:, h * group:(h + 1) * group] = torch.einsum("sngk,kd->sngd", torch.softmax(s, 3), vv).reshape(-1, group, D)
    assert float((got.double() - want).norm() / want.norm()) < BOUND[dtype]
