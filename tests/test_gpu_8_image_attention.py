"""The image-token attention operators on the GPU against their formulas in 64 bits (image_attention_ref): norm and
rotation of packed projections, the choice of key blocks, attention over them, and the three as one layer."""
import ctypes
import importlib.util

import numpy as np
import pytest

import image_attention_ref as ref
from conftest import max_rel_err

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]


def up(ctx, a):
    return ctx.upload(a, dtype=a.dtype)


def close(got, want, tol):
    got = ref.wide(got)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.max((np.abs(got - want) / tol)[bad])), np.argwhere(bad)[:4])


# ------------------------------------------------------------------------------------------------ norm and rotation

def rope_tolerance(y, size, kind):
    """24 roundings of 2^-24 of the pair's length: the mean of squares (8 + 5), root, quotient, gamma, the angle's
    reduction (3) and its cosine and sine (2), the turn (3); then the result's own rounding."""
    f32 = 24 * 2.0 ** -24 * size
    return f32 + ref.HALF_STEP[kind] * (np.abs(y) + f32) + ref.TINY[kind]


ROPE = [  # n, tokens, heads, kv_heads, dim, axis_dims, halves, norm, far, x kind, out kind, stride beyond the row
    (1, 1, 1, 1, 8, (0, 4, 4), False, True, 0, "f32", "f32", 0),
    (2, 7, 3, 3, 40, (0, 20, 20), False, True, 30, "f32", "f16", 0),
    (2, 130, 8, 2, 40, (0, 20, 20), True, True, 30, "f32", "bf16", 8),
    (1, 33, 2, 1, 128, (16, 56, 56), False, True, 1000, "bf16", "bf16", 64),
    (1, 33, 2, 1, 128, (16, 56, 56), True, True, 1000, "f16", "f16", 0),
    (3, 65, 10, 5, 80, (6, 10, 50), True, False, 1_000_000, "f32", "f32", 4),
    (3, 65, 10, 5, 80, (6, 10, 50), False, False, 1_000_000, "f32", "f32", 0),
    (1, 9, 40, 1, 256, (64, 96, 96), True, True, 100, "f32", "f32", 0),
    (1, 1, 33, 3, 72, (0, 0, 72), False, True, 100, "f16", "f16", 0),
    (1, 300, 1, 1, 24, (2, 2, 2), True, True, 100, "bf16", "bf16", 8),
    (2, 2500, 8, 8, 64, (0, 32, 32), False, True, 100, "f32", "f16", 0)]


@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_qkv_norm_rope(mbx, ctx, case):
    n, tokens, heads, kv, dim, axis_dims, halves, norm, far, x_kind, kind, beyond = case
    rng = np.random.default_rng(dim + tokens)
    row = (heads + 2 * kv) * dim
    x = ref.narrow(rng.standard_normal((n, tokens, row + beyond)) * 3, x_kind)
    items = n if far > 50 else 1
    pos = (rng.integers(0, far + 1, (items, tokens, 3)) + rng.integers(0, 2, (items, tokens, 3)) * 0.25)
    pos = pos.astype(np.float32)
    gq, gk = (rng.normal(1, 0.2, dim).astype(np.float32) for _ in range(2))
    out = mbx.qkv_norm_rope(up(ctx, x), heads, kv, dim, positions=up(ctx, pos), axis_dims=axis_dims, theta=1000.0,
                            pairing="halves" if halves else "adjacent", norm=norm, q_gamma=up(ctx, gq),
                            k_gamma=up(ctx, gk), eps=1e-5, dtype=ref.KINDS[kind])
    parts = ref.wide(x)[..., :row].reshape(n, tokens, heads + 2 * kv, dim)
    for got, part, gamma in ((out[0], parts[:, :, :heads], gq), (out[1], parts[:, :, heads:heads + kv], gk)):
        y, size = ref.norm_rope(part, gamma, 1e-5, norm, pos, axis_dims, 1000.0, halves)
        close(got.numpy(), y, rope_tolerance(y, size, kind))
    close(out[2].numpy(), parts[:, :, heads + kv:], ref.HALF_STEP[kind] * np.abs(parts[:, :, heads + kv:])
          + ref.TINY[kind])


# From 128 tokens an SM on, a warp takes a second token. x ends with the last token's row, and a warp's
# step holds up to 32 / (dim / 8) heads, more than the token has in the first four.
ROPE_LONG = [
    (1, 18947, 1, 1, 40, (0, 20, 20), True, True, 30, "f32", "f16", 0),
    (3, 6400, 1, 1, 64, (0, 32, 32), False, True, 100, "bf16", "bf16", 0),
    (1, 20001, 6, 1, 24, (2, 10, 12), True, True, 30, "f32", "bf16", 0),
    (1, 18961, 2, 0, 8, (0, 4, 4), False, False, 30, "f16", "f16", 0),
    (1, 18955, 3, 1, 128, (16, 56, 56), True, True, 30, "f16", "f16", 0),
    (2, 9500, 9, 3, 72, (0, 36, 36), False, True, 100, "f32", "f32", 4)]


@pytest.mark.parametrize("case", ROPE_LONG, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_qkv_norm_rope_of_two_tokens_a_warp(mbx, ctx, case):
    test_qkv_norm_rope(mbx, ctx, case)


def test_qkv_norm_rope_parts(mbx, ctx):
    """q alone, k alone, no v (whose part of the row does not exist then), no positions, no gamma."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 11, 3 * 16)).astype(np.float32)
    parts = x.astype(np.float64).reshape(2, 11, 3, 16)
    want, size = ref.norm_rope(parts, None, 1e-6, True, None, (0, 0, 0), 1.0, False)
    tol = rope_tolerance(want, size, "f32")
    d = up(ctx, x)
    q = ctx.empty((2, 11, 3, 16))
    mbx.qkv_norm_rope(d, 3, 0, 16, out=(q, None, None))
    close(q.numpy(), want, tol)
    k = ctx.empty((2, 11, 3, 16))
    mbx.qkv_norm_rope(d, 0, 3, 16, out=(None, k, None))
    close(k.numpy(), want, tol)
    q, k = ctx.empty((2, 11, 2, 16)), ctx.empty((2, 11, 1, 16))
    mbx.qkv_norm_rope(d, 2, 1, 16, out=(q, k, None))
    close(q.numpy(), want[:, :, :2], tol[:, :, :2])
    close(k.numpy(), want[:, :, 2:], tol[:, :, 2:])
    plain = mbx.qkv_norm_rope(d, 1, 1, 16, norm=False)
    for got, i in zip(plain, range(3)):
        assert np.array_equal(got.numpy()[:, :, 0], x.reshape(2, 11, 3, 16)[:, :, i])
    empty = mbx.qkv_norm_rope(ctx.empty((2, 0, 48)), 1, 1, 16)
    assert [t.shape for t in empty] == [(2, 0, 1, 16)] * 3


@pytest.mark.parametrize("dim", [24, 40, 64, 72, 80, 104, 200])
def test_qkv_norm_rope_has_one_factor_a_head(mbx, ctx, dim):
    """The norm's factor is the head's: every eighth channel is 1 here, so it is the factor itself."""
    rng = np.random.default_rng(dim)
    x = rng.standard_normal((1, 500, 3, dim)).astype(np.float32)
    x[..., ::8] = 1.0
    q, k, _ = mbx.qkv_norm_rope(up(ctx, x.reshape(1, 500, 3 * dim)), 1, 1, dim)
    for got in (q.numpy(), k.numpy()):
        factors = got[..., ::8]
        assert (factors == factors[..., :1]).all()


def test_qkv_norm_rope_keeps_nan_in_its_head(mbx, ctx):
    x = np.ones((1, 3, 4 * 8), np.float32)
    x[0, 1, 8] = np.nan
    pos = np.zeros((3, 3), np.float32)
    pos[2] = np.inf
    q, k, v = (t.numpy() for t in mbx.qkv_norm_rope(up(ctx, x), 2, 1, 8, positions=up(ctx, pos), axis_dims=(0, 4, 0)))
    assert np.isnan(q[0, 1, 1]).all() and not np.isnan(q[0, 1, 0]).any() and not np.isnan(k[0, 1]).any()
    assert np.isnan(q[0, 2, :, :4]).all() and not np.isnan(q[0, 2, :, 4:]).any()  # a position that is no number
    assert not np.isnan(q[0, 0]).any() and not np.isnan(v).any()


# ------------------------------------------------------------------------------------------------ choice of blocks

def tokens_field(rng, n, tokens, heads, dim, run=40):
    x = np.repeat(rng.standard_normal((n, tokens // run + 1, heads, dim)), run, axis=1)[:, :tokens]
    return x + 0.5 * rng.standard_normal((n, tokens, heads, dim))


def key_mask(rng, n, nk, how):
    if how == "none":
        return None
    m = (rng.random((n, nk)) < 0.8).astype(np.uint8) * 3
    m[:, nk // 4:nk // 2] = 0
    if how == "empty":
        m[-1] = 0
    return m


SELECT = [  # n, nq, nk, heads, kv_heads, dim, block_k, topk, mask, kind
    (1, 1, 1, 1, 1, 8, 16, 1, "none", "f32"), (1, 1, 1, 1, 1, 8, 16, 3, "empty", "f16"),
    (2, 129, 300, 4, 2, 40, 16, 5, "empty", "f32"), (1, 128, 4096, 2, 2, 64, 64, 7, "none", "bf16"),
    (3, 257, 1000, 6, 1, 128, 128, 8, "hole", "f16"), (1, 700, 5000, 3, 3, 256, 32, 100, "hole", "bf16"),
    (2, 1000, 900, 5, 5, 72, 64, 20, "hole", "f32"), (1, 9000, 9000, 2, 1, 24, 16, 33, "none", "f16"),
    (1, 127, 20000, 1, 1, 16, 16, 640, "none", "f32")]


@pytest.mark.parametrize("case", SELECT, ids=lambda c: "-".join(map(str, c)))
def test_block_select(mbx, ctx, case):
    n, nq, nk, heads, kv, dim, block_k, topk, how, kind = case
    rng = np.random.default_rng(nk + dim)
    q, k = (ref.narrow(tokens_field(rng, n, t, h, dim), kind) for t, h in ((nq, heads), (nk, kv)))
    mask = key_mask(rng, n, nk, how)
    if mask is not None:  # what a mask hides may hold anything
        poison = ref.narrow(np.full(k.shape, np.nan), kind)
        k = np.where((mask == 0)[:, :, None, None], poison, k)
    got = mbx.block_select(up(ctx, q), up(ctx, k), topk, block_k=block_k,
                           key_mask=None if mask is None else up(ctx, mask)).numpy()
    assert np.array_equal(got, ref.select(ref.wide(q), ref.wide(k), topk, block_k, mask))


def test_block_select_ties_and_special_scores(mbx, ctx):
    """Equal scores go to the lower block, +0 and -0 are equal, NaN is above everything, -inf below, but above a block
    without a key."""
    k = np.zeros((1, 16 * 8, 1, 8), np.float32)
    q = np.zeros((1, 5, 1, 8), np.float32)
    q[..., 0] = 1.0
    level = np.float32([0.0, 2.0, -0.0, np.nan, -np.inf, 2.0, 0.0, 9.0])
    k[0, :, 0, 0] = np.repeat(level, 16)
    mask = np.ones((1, 128), np.uint8)
    mask[0, 112:] = 0
    want = {1: [3], 2: [1, 3], 3: [1, 3, 5], 4: [0, 1, 3, 5], 5: [0, 1, 2, 3, 5], 6: [0, 1, 2, 3, 5, 6],
            7: [0, 1, 2, 3, 4, 5, 6], 9: [0, 1, 2, 3, 4, 5, 6, -1, -1]}
    for topk, blocks in want.items():
        got = mbx.block_select(up(ctx, q), up(ctx, k), topk, block_k=16, key_mask=up(ctx, mask)).numpy()
        assert got[0, 0, 0].tolist() == blocks
    same = np.ones((1, 64 * 40, 1, 8), np.float32)
    got = mbx.block_select(up(ctx, q), up(ctx, same), 17, block_k=64).numpy()
    assert got[0, 0, 0].tolist() == list(range(17))


def test_block_select_of_no_keys(mbx, ctx):
    q, k = ctx.upload(np.ones((2, 130, 2, 8))), ctx.empty((2, 0, 1, 8))
    assert (mbx.block_select(q, k, 3).numpy() == -1).all()


# ------------------------------------------------------------------------------------------------ attention

ATTEND = [  # n, nq, nk, heads, kv_heads, dim, block_k, topk, mask
    (1, 1, 1, 1, 1, 8, 16, 1, "none"), (2, 1, 777, 4, 2, 64, 64, 9, "none"), (1, 3, 5000, 2, 1, 128, 32, 60, "hole"),
    (2, 127, 130, 2, 2, 40, 16, 4, "empty"), (1, 128, 128, 3, 1, 128, 128, 1, "none"),
    (1, 129, 513, 2, 2, 80, 128, 3, "hole"), (3, 200, 1000, 4, 4, 16, 64, 5, "empty"),
    (1, 400, 2000, 6, 2, 128, 64, 16, "none"), (2, 300, 700, 2, 1, 72, 32, 13, "hole"),
    (1, 1030, 1030, 1, 1, 120, 16, 20, "hole"), (1, 513, 4096, 2, 2, 64, 128, 32, "none"),
    (1, 5, 300, 1, 1, 56, 16, 25, "none"), (1, 130, 200, 1, 1, 8, 16, 5, "none"), (2, 260, 999, 3, 3, 24, 32, 31, "hole"),
    (1, 129, 300, 2, 1, 104, 64, 9, "empty"), (1, 130, 20000, 1, 1, 16, 16, 1100, "none"),
    (1, 1, 20000, 1, 1, 16, 16, 1100, "hole")]


def attend_inputs(rng, n, nq, nk, heads, kv, dim, block_k, topk, how, kind):
    q = ref.narrow(tokens_field(rng, n, nq, heads, dim), kind)
    k, v = (ref.narrow(tokens_field(rng, n, nk, kv, dim), kind) for _ in range(2))
    mask = key_mask(rng, n, nk, how)
    if mask is not None:
        hidden = (mask == 0)[:, :, None, None]
        k = np.where(hidden, ref.narrow(np.full(k.shape, np.nan), kind), k)
        v = np.where(hidden, ref.narrow(np.full(k.shape, np.inf), kind), v)
    blocks = -(-nk // block_k)
    index = np.full((n, heads, -(-nq // 128), topk), -1, np.int32)
    for at in np.ndindex(index.shape[:3]):
        chosen = np.sort(rng.permutation(blocks)[:topk])
        index[at][:len(chosen)] = chosen
    return q, k, v, mask, index


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c)))
def test_block_attention(mbx, ctx, case, kind):
    rng = np.random.default_rng(case[2] + case[5])
    q, k, v, mask, index = attend_inputs(rng, *case, kind)
    out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)), block_k=case[6],
                              key_mask=None if mask is None else up(ctx, mask))
    want, tol = ref.attention(*(ref.wide(t) for t in (q, k, v)), index, case[6], mask, case[5] ** -0.5, kind)
    close(out.numpy(), want, tol)


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("nq", [2, 150])
def test_block_attention_takes_any_index(mbx, ctx, kind, nq):
    """Entries outside the blocks are skipped wherever they stand, a block listed twice counts twice, and a list
    without any block leaves zeros."""
    rng = np.random.default_rng(5)
    q, k, v, _, _ = attend_inputs(rng, 1, nq, 200, 2, 1, 48, 64, 2, "none", kind)
    index = np.full((1, 2, -(-nq // 128), 9), -1, np.int32)
    index[0, 0, 0] = [3, -1, 0, 4, 3, -2147483648, 2147483647, 0, 0]
    index[0, 1, 0] = [-7, 4, 5, 100, -1, -1, -1, -1, 2]
    out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)))
    want, tol = ref.attention(*(ref.wide(t) for t in (q, k, v)), index, 64, None, 48 ** -0.5, kind)
    close(out.numpy(), want, tol)
    if nq > 128:
        assert not ref.wide(out.numpy())[:, 128:].any()


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("nq", [1, 140])
def test_block_attention_of_no_keys(mbx, ctx, kind, nq):
    q = up(ctx, ref.narrow(np.ones((2, nq, 2, 16)), kind))
    none = up(ctx, ref.narrow(np.ones((2, 0, 1, 16)), kind))
    some = up(ctx, ref.narrow(np.ones((2, 33, 1, 16)), kind))
    blocks = -(-nq // 128)
    for k, topk in ((none, 2), (none, 0), (some, 0)):
        index = ctx.upload(np.zeros((2, 2, blocks, topk)), dtype=np.int32)
        out = up(ctx, ref.narrow(np.full((2, nq, 2, 16), 7.0), kind))
        assert not ref.wide(mbx.block_attention(q, k, k, index, out=out).numpy()).any()


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("nq", [1, 140])
def test_block_attention_wide_logits(mbx, ctx, kind, nq):
    """Logits from very negative to very positive, growing along the list, so that the running maximum keeps moving;
    the lowest value of the type and a scale of either sign."""
    rng = np.random.default_rng(11)
    q, k, v, _, index = attend_inputs(rng, 1, nq, 640, 2, 2, 64, 64, 10, "none", kind)
    k = ref.narrow(ref.wide(k) * np.linspace(0.1, 6.0, 640)[None, :, None, None], kind)
    for scale in (0.5, -0.5, 0.0):
        out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)), scale=scale)
        want, tol = ref.attention(*(ref.wide(t) for t in (q, k, v)), index, 64, None, scale, kind)
        close(out.numpy(), want, tol)


@pytest.mark.parametrize("kind,size", [("f32", 1e-4), ("f32", 1e3), ("bf16", 1e-4), ("bf16", 1e3), ("f16", 1e-4),
                                       ("f16", 20.0)])  # f16 holds 1500 standard deviations times 20, not times 1e3
def test_block_attention_of_small_and_large_values(mbx, ctx, kind, size):
    """Values far from one, with a channel and a token far above the others."""
    rng = np.random.default_rng(13)
    q, k, v, _, index = attend_inputs(rng, 1, 140, 300, 2, 1, 40, 32, 6, "none", kind)
    far = ref.wide(v) * size
    far[:, :, :, 3] *= 30
    far[:, 17] *= 10
    v = ref.narrow(far, kind)
    k = ref.narrow(ref.wide(k) * size, kind)
    out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)), block_k=32, scale=0.2 / size)
    want, tol = ref.attention(*(ref.wide(t) for t in (q, k, v)), index, 32, None, 0.2 / size, kind)
    close(out.numpy(), want, tol)


def exact_weights(rng, nq, nk, heads, dim):
    """q and k whose logits are whole numbers, exact in any summation: 0 or -200 by the key's first channel."""
    q, k = np.zeros((1, nq, heads, dim), np.float32), np.zeros((1, nk, 1, dim), np.float32)
    q[..., 0] = 1.0
    return q, k, rng.standard_normal((1, nk, 1, dim)).astype(np.float32)


def equal_weights_tolerance(v, keys):
    """Of the mean of v over `keys`, in units of its mean magnitude (weights are exactly 1 there): a value's two parts
    2^-22; at most 128 keys in an unbroken sum, 8 steps of 16 keys in three products each, 2^-23 a step; their joining,
    the sum of weights and the quotient, 8 roundings of 2^-24."""
    return (2.0 ** -22 + 24 * 2.0 ** -23 + 8 * 2.0 ** -24) * np.abs(v[0, keys, 0].astype(np.float64)).mean(0)


@pytest.mark.parametrize("heads", [2, 148])  # lists that are split over CTAs, and whole ones
@pytest.mark.parametrize("nq", [2, 140])
@pytest.mark.parametrize("typical,far", [(1.0, 4.0), (1e-4, 0.1), (1e-5, 1.0), (1.0, 1e9), (1.0, 1e30), (1e-20, 1.0)])
def test_f32_attention_does_not_depend_on_other_blocks_values(mbx, ctx, typical, far, nq, heads):
    """Neither a row of a block that no list names nor a listed one of no weight costs the others their bits."""
    rng = np.random.default_rng(41)
    nk, dim = 640, 24
    q, k, v = exact_weights(rng, nq, nk, heads, dim)
    v *= typical
    v[0, 37] = far      # block 0, unlisted
    k[0, 37] = far
    v[0, 38], k[0, 39] = np.nan, np.inf
    v[0, 330:336] = far  # block 5, listed; no weight
    k[0, 320:384, 0, 0] = -200.0
    lists = [1, 2, 3, 5, 7, 8]
    index = np.broadcast_to(np.int32(lists), (1, heads, -(-nq // 128), len(lists))).copy()
    out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)), scale=1.0).numpy()
    keys = np.concatenate([np.arange(b * 64, b * 64 + 64) for b in lists if b != 5])
    want = v[0, keys, 0].astype(np.float64).mean(0)
    tol = equal_weights_tolerance(v, keys) + far * np.exp(-200.0)
    close(out, np.broadcast_to(want, out.shape), np.broadcast_to(tol, out.shape))


@pytest.mark.parametrize("heads", [2, 148])
def test_f32_attention_of_blocks_of_every_magnitude(mbx, ctx, heads):
    """Each 16 keys have values of another magnitude, zero among them, and keys of another one too."""
    rng = np.random.default_rng(43)
    nq, nk, dim = 140, 960, 16
    for powers in ([-120, -20, 0, 20, 120], [-140, -130, -126], [0, 0, -400]):  # -400: zero
        q, k, v = (rng.standard_normal((1, t, h, dim)) for t, h in ((nq, heads), (nk, 1), (nk, 1)))
        size = 2.0 ** rng.choice(powers, nk // 16).repeat(16)
        v = (v * size[None, :, None, None]).astype(np.float32)
        k = (k * (2.0 ** rng.integers(-12, 3, nk // 16).repeat(16))[None, :, None, None]).astype(np.float32)
        turn = 2.0 ** 100 if powers[0] == 0 else 1.0  # magnitudes of q and k that their products do not have
        q, k = (q / turn).astype(np.float32), (k * turn).astype(np.float32)
        index = np.full((1, heads, 2, 30), -1, np.int32)
        for at in np.ndindex(index.shape[:3]):
            index[at][:25] = np.sort(rng.permutation(30)[:25])
        out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)), block_k=32, scale=0.5)
        want, tol = ref.attention(*(ref.wide(t) for t in (q, k, v)), index, 32, None, 0.5, "f32")
        # Below 2^-126 a rounding is off by up to 2^-150: 13 shares of the list (25 blocks of 32 keys in tiles of 64), each
        # rounded, weighted by at most one and added with a rounding, over a sum of weights of at least 1/2 (the largest
        # share's reference is its maximum rounded up to a whole log2): 26 * 2^-150 * 2 + 2^-150 < 2^-144.
        close(out.numpy(), want, tol + 2.0 ** -144)


def test_block_attention_long_list_of_one_token(mbx, ctx):
    """More list entries for one CTA than it keeps in shared memory at a time."""
    rng = np.random.default_rng(31)
    heads, blocks, dim = 40, 12000, 8
    q, k, v = (ref.narrow(rng.standard_normal((1, t, h, dim)), "f16") for t, h in
               ((1, heads), (blocks * 16, 1), (blocks * 16, 1)))
    index = np.broadcast_to(np.arange(blocks, dtype=np.int32), (1, heads, 1, blocks)).copy()
    index[0, :, 0, 5000:7000] = -1
    out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)), block_k=16)
    wide = [ref.wide(t) for t in (q, k, v)]
    kept = np.r_[0:5000 * 16, 7000 * 16:blocks * 16]
    p = np.exp(wide[0][0, 0] @ wide[1][0, kept, 0].T * dim ** -0.5)
    total = p.sum(1, keepdims=True)
    want, spread = p @ wide[2][0, kept, 0] / total, p @ np.abs(wide[2][0, kept, 0]) / total
    # f32 throughout: at most 12000 roundings of 2^-24 in a lane's sums, 2^-17 for logits and exponentials.
    tol = (12000 * 2.0 ** -24 + 2.0 ** -17) * spread
    close(out.numpy()[0, 0], want, tol + ref.HALF_STEP["f16"] * (np.abs(want) + tol))


@pytest.mark.parametrize("dim", [8, 72])
def test_block_attention_long_list_of_many_rows(mbx, ctx, dim):
    """Equal weights over two million keys: the tensor core truncates its sums, which must not show in the mean.

    Positive values, so that truncations add up: 2048 steps of 16 keys in an unbroken sum, in two additions each that
    lose up to 2^-23; joining, the sum of weights and the quotient 2^-16; the result's rounding."""
    rng = np.random.default_rng(47)
    heads, nq, nk, block_k = 150, 129, 1 << 21, 128  # 300 query blocks fill the card: lists need not be split
    v = (0.5 + 0.5 * rng.random((1, nk, 1, dim))).astype(np.float16)
    index = np.broadcast_to(np.arange(nk // block_k, dtype=np.int32), (1, heads, 2, nk // block_k))
    q, d = up(ctx, np.zeros((1, nq, heads, dim), np.float16)), up(ctx, v)
    out = mbx.block_attention(q, d, d, up(ctx, np.ascontiguousarray(index)), block_k=block_k).numpy()
    want = np.broadcast_to(v[0, :, 0].astype(np.float64).mean(0), out.shape)
    close(out, want, (2048 * 2.0 ** -22 + 2.0 ** -16 + 2.0 ** -11) * want)
    ctx.synchronize()
    ctx.release_below(1 << 62)


@pytest.mark.parametrize("kind,nq", [("f32", 1), ("f16", 1), ("bf16", 200)])
def test_offsets_past_32_bits(mbx, ctx, kind, nq):
    """Keys and values in rows of 1024 elements, over two million tokens on: element offsets past 2^31."""
    rng = np.random.default_rng(37)
    row, dim, nk, last = 1024, 64, 2_200_000, 3
    step = ref.KINDS[kind].itemsize
    big = ctx.alloc(nk * row * step)
    try:
        block = 64
        first = nk // block - last  # the last full blocks
        kv = [ref.narrow(rng.standard_normal((last * block, dim)), kind) for _ in range(2)]
        rows = np.zeros((last * block, row), ref.KINDS[kind])
        rows[:, 128:128 + dim], rows[:, 512:512 + dim] = kv
        at = big + first * block * row * step
        mbx.check(mbx.abi.lib().mbx_memcpy_h2d(ctx.handle, at, rows.ctypes.data_as(ctypes.c_void_p), rows.nbytes))
        ctx.synchronize()
        q = ref.narrow(rng.standard_normal((1, nq, 1, dim)), kind)
        k, v = (mbx.DeviceTensor.wrap(ctx, big + c * step, (1, nk, 1, dim), ref.KINDS[kind]) for c in (128, 512))
        index = np.broadcast_to(np.arange(first, first + last, dtype=np.int32), (1, 1, -(-nq // 128), last)).copy()
        out = mbx.block_attention(up(ctx, q), k, v, up(ctx, index), k_stride=row, v_stride=row)
        want, tol = ref.attention(ref.wide(q), *(ref.wide(t)[None, :, None] for t in kv), index - first, 64, None,
                                  dim ** -0.5, kind)
        close(out.numpy(), want, tol)
    finally:
        ctx.synchronize()
        ctx.free(big)
        ctx.release_below(1 << 62)


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("nq", [2, 200])
def test_packed_rows_serve_in_place(mbx, ctx, kind, nq):
    """q, k and v as parts of one wider row, and rows behind the tensors left as they were."""
    rng = np.random.default_rng(7)
    heads, kv, dim, n = 4, 2, 24, 2
    row = (heads + 2 * kv) * dim + 16
    x = ref.narrow(rng.standard_normal((n, nq, row)), kind)
    d = up(ctx, x)
    step = x.dtype.itemsize
    q, k, v = (mbx.DeviceTensor.wrap(ctx, d.ptr + at * dim * step, (n, nq, h, dim), x.dtype)
               for at, h in ((0, heads), (heads, kv), (heads + kv, kv)))
    index = mbx.block_select(q, k, 3, block_k=16, q_stride=row, k_stride=row)
    w = ref.wide(x)[..., :row - 16].reshape(n, nq, heads + 2 * kv, dim)
    wq, wk, wv = w[:, :, :heads], w[:, :, heads:heads + kv], w[:, :, heads + kv:]
    assert np.array_equal(index.numpy(), ref.select(wq, wk, 3, 16))
    wide_out = up(ctx, ref.narrow(np.full((n * nq + 5, heads, dim), 7.0), kind))
    out = mbx.DeviceTensor.wrap(ctx, wide_out.ptr, (n, nq, heads, dim), x.dtype)
    mbx.block_attention(q, k, v, index, block_k=16, q_stride=row, k_stride=row, v_stride=row, out=out)
    want, tol = ref.attention(wq, wk, wv, index.numpy(), 16, None, dim ** -0.5, kind)
    all_rows = wide_out.numpy()
    close(all_rows[:n * nq].reshape(want.shape), want, tol)
    assert (ref.wide(all_rows[n * nq:]) == 7.0).all()


@pytest.mark.parametrize("kind", DTYPES)
def test_twice_the_same_bits(mbx, ctx, kind):
    rng = np.random.default_rng(19)
    for nq in (1, 300):
        q, k, v, mask, index = attend_inputs(rng, 2, nq, 3000, 2, 1, 64, 64, 30, "hole", kind)
        d = [up(ctx, t) for t in (q, k, v, index)]
        m = up(ctx, mask)
        first = mbx.block_attention(*d, key_mask=m).numpy()
        assert all(mbx.block_attention(*d, key_mask=m).numpy().tobytes() == first.tobytes() for _ in range(3))


# ------------------------------------------------------------------------------------------------ as they are used

def layer(mbx, x, w_qkv, w_out, pos, mask, heads, kv, dim, kind):
    """One attention layer over image tokens: projection, heads, choice, attention, projection with residual."""
    n, h, w, c = x.shape
    qkv = mbx.conv1x1(x, w_qkv)
    rows = mbx.DeviceTensor.wrap(x.ctx, qkv.ptr, (n, h * w, w_qkv.c_out))
    q, k, v = mbx.qkv_norm_rope(rows, heads, kv, dim, positions=pos, axis_dims=(0, dim // 2, dim // 2),
                                dtype=ref.KINDS[kind])
    index = mbx.block_select(q, k, 4, block_k=32, key_mask=mask)
    o = mbx.block_attention(q, k, v, index, block_k=32, key_mask=mask)
    out = None
    if kind == "f32":
        out = mbx.conv1x1(mbx.DeviceTensor.wrap(x.ctx, o.ptr, (n, h, w, heads * dim)), w_out, residual=x)
    return qkv, q, k, v, index, o, out


@pytest.mark.parametrize("kind", DTYPES)
def test_the_operators_together(mbx, ctx, oracle, kind):
    rng = np.random.default_rng(23)
    n, h, w, c, heads, kv, dim = 2, 13, 25, 64, 4, 2, 32
    x = rng.standard_normal((n, h, w, c)).astype(np.float32)
    wq = (rng.standard_normal(((heads + 2 * kv) * dim, c)) / 8).astype(np.float32)
    wo = (rng.standard_normal((c, heads * dim)) / 11).astype(np.float32)
    pos = np.stack(np.meshgrid([0], np.arange(h), np.arange(w), indexing="ij"), -1).reshape(-1, 3).astype(np.float32)
    mask = key_mask(rng, n, h * w, "hole")
    pq, po = mbx.Param(ctx, wq), mbx.Param(ctx, wo)
    d = up(ctx, x)
    qkv, q, k, v, index, o, out = layer(mbx, d, pq, po, up(ctx, pos), up(ctx, mask), heads, kv, dim, kind)
    rows = qkv.numpy().astype(np.float64).reshape(n, h * w, -1, dim)
    for got, part in ((q, rows[:, :, :heads]), (k, rows[:, :, heads:heads + kv])):
        y, size = ref.norm_rope(part, None, 1e-6, True, pos[None], (0, 16, 16), 10000.0, False)
        close(got.numpy(), y, rope_tolerance(y, size, kind))
    q, k, v = (ref.wide(t.numpy()) for t in (q, k, v))
    assert np.array_equal(index.numpy(), ref.select(q, k, 4, 32, mask))
    want, tol = ref.attention(q, k, v, index.numpy(), 32, mask, dim ** -0.5, kind)
    close(o.numpy(), want, tol)
    if out is not None:
        want = oracle.conv1x1(o.numpy().reshape(n, h, w, -1), wo, None, x)
        assert max_rel_err(out.numpy(), want) <= 1e-5
    pq.close()
    po.close()


@pytest.mark.skipif(importlib.util.find_spec("torch") is None, reason="captures with torch")
@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("nq", [1, 200])
def test_two_captured_calls_at_once(mbx, kind, nq):
    """Two graphs with a workspace each, replayed side by side on two streams, on new inputs in the same buffers."""
    import torch
    rng = np.random.default_rng(29)
    with mbx.Context(0) as ctx:
        sides = []
        for side in range(2):
            q, k, v, _, index = attend_inputs(rng, 1, nq, 2000, 2, 1, 64, 32, 20, "none", kind)
            t = dict(q=up(ctx, q), k=up(ctx, k), v=up(ctx, v), index=up(ctx, index), out=up(ctx, q))
            t["ws"] = mbx.block_attention_workspace(t["q"], t["k"], t["index"], block_k=32)
            t["select_ws"] = mbx.block_select_workspace(t["q"], t["k"], block_k=32)
            sides.append(t)
        ctx.synchronize()
        graphs = []
        for t in sides:
            stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

            def call():
                ctx.set_stream(stream.cuda_stream)
                mbx.block_select(t["q"], t["k"], 20, block_k=32, workspace=t["select_ws"], out=t["index"])
                mbx.block_attention(t["q"], t["k"], t["v"], t["index"], block_k=32, workspace=t["ws"], out=t["out"])
            call()
            ctx.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                call()
            graphs.append((graph, stream))
            ctx.set_stream(None)
        new = [attend_inputs(rng, 1, nq, 2000, 2, 1, 64, 32, 20, "none", kind)[:3] for _ in sides]
        for t, arrays in zip(sides, new):
            for name, a in zip("qkv", arrays):
                mbx.check(mbx.abi.lib().mbx_memcpy_h2d(ctx.handle, t[name].vp, a.ctypes.data_as(ctypes.c_void_p),
                                                       a.nbytes))
        ctx.synchronize()
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in graphs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for t, arrays in zip(sides, new):
            wide = [ref.wide(a) for a in arrays]
            index = t["index"].numpy()
            assert np.array_equal(index, ref.select(wide[0], wide[1], 20, 32))
            want, tol = ref.attention(*wide, index, 32, None, 0.125, kind)
            close(t["out"].numpy(), want, tol)
        del graphs


def test_pool_keeps_streams_apart(mbx):
    """A block freed on one stream may still be in use there: another stream gets it only after a synchronize."""
    legacy = 1  # the legacy default stream's handle
    with mbx.Context(0) as ctx:
        def block():
            t = ctx.empty((1 << 20,))
            t.free_at = t.ptr
            return t
        first = block()
        first.free()
        ctx.set_stream(legacy)
        second = block()
        assert second.ptr != first.free_at
        second.free()
        ctx.set_stream(None)
        again = block()
        assert again.ptr == first.free_at  # its own stream's order is enough
        again.free()
        ctx.synchronize()
        ctx.set_stream(legacy)
        both = [block(), block()]
        assert {t.ptr for t in both} == {first.free_at, second.free_at}


@pytest.mark.skipif(importlib.util.find_spec("torch") is None, reason="captures with torch")
def test_a_captured_call_needs_its_own_workspace(mbx):
    import torch
    with mbx.Context(0) as ctx:
        q = ctx.upload(np.ones((1, 200, 2, 16)), dtype=np.float16)
        index, out = mbx.block_select(q, q, 2), ctx.empty(q.shape, q.dtype)
        mbx.block_attention(q, q, q, index, out=out)
        ctx.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        assert not ctx.capturing
        with torch.cuda.graph(graph, stream=stream):
            ctx.set_stream(stream.cuda_stream)
            assert ctx.capturing
            with pytest.raises(ValueError, match="workspace"):
                mbx.block_select(q, q, 2, out=index)
            with pytest.raises(ValueError, match="workspace"):
                mbx.block_attention(q, q, q, index, out=out)
        ctx.set_stream(None)
        assert not ctx.capturing
        del graph


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("nq,heads", [(1, 1), (1, 70), (140, 2), (140, 148)])  # rows, split rows, split and whole lists
def test_block_attention_to_float32(mbx, ctx, kind, nq, heads):
    """The result of any operands before it is rounded to their type, and zeros where no key is."""
    rng = np.random.default_rng(53)
    q, k, v, mask, index = attend_inputs(rng, 2, nq, 500, heads, 1, 40, 32, 9, "empty", kind)
    out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)), block_k=32, key_mask=up(ctx, mask),
                              out_dtype=np.float32)
    assert out.dtype == np.float32
    want, tol = ref.attention(*(ref.wide(t) for t in (q, k, v)), index, 32, mask, 40 ** -0.5, kind)
    # Less the rounding that ref.attention counts for the operands' type, (|o| + t) of HALF_STEP, and with f32's.
    half = ref.HALF_STEP[kind]
    tol = (tol - ref.TINY[kind] - half * np.abs(want)) / (1 + half)
    close(out.numpy(), want, np.maximum(tol, 0) + 2.0 ** -24 * np.abs(want) + ref.TINY["f32"])
    none = ctx.empty((2, 0, 1, 40), q.dtype)
    index = up(ctx, np.zeros((2, heads, -(-nq // 128), 1), np.int32))
    given = up(ctx, np.full(q.shape, 7.0, np.float32))
    assert not mbx.block_attention(up(ctx, q), none, none, index, out=given).numpy().any()


@pytest.mark.parametrize("kind", DTYPES)
def test_the_operators_between_two_projections(mbx, ctx, oracle, kind):
    """From one 1x1 convolution to the next in every type: the attention hands float32 on."""
    rng = np.random.default_rng(59)
    n, h, w, c, heads, dim = 1, 12, 20, 64, 4, 32
    x = rng.standard_normal((n, h, w, c)).astype(np.float32)
    weights = [(rng.standard_normal(s) / 9).astype(np.float32) for s in ((3 * heads * dim, c), (c, heads * dim))]
    p_in, p_out = (mbx.Param(ctx, t) for t in weights)
    d = up(ctx, x)
    qkv = mbx.conv1x1(d, p_in)
    rows = mbx.DeviceTensor.wrap(ctx, qkv.ptr, (n, h * w, p_in.c_out))
    q, k, v = mbx.qkv_norm_rope(rows, heads, heads, dim, dtype=ref.KINDS[kind])
    index = mbx.block_select(q, k, 5, block_k=32)
    o = mbx.block_attention(q, k, v, index, block_k=32, out_dtype=np.float32)
    y = mbx.conv1x1(mbx.DeviceTensor.wrap(ctx, o.ptr, (n, h, w, heads * dim)), p_out, residual=d)
    want = oracle.conv1x1(o.numpy().reshape(n, h, w, -1), weights[1], None, x)
    assert max_rel_err(y.numpy(), want) <= 1e-5
    attended, tol = ref.attention(*(ref.wide(t.numpy()) for t in (q, k, v)), index.numpy(), 32, None, dim ** -0.5, kind)
    close(o.numpy(), attended, tol)
    p_in.close()
    p_out.close()


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("nk", [1, 2, 15, 17])
def test_block_attention_of_few_keys_for_many_rows(mbx, ctx, kind, nk):
    rng = np.random.default_rng(61)
    for dim in (40, 96):
        q, k, v, _, index = attend_inputs(rng, 2, 200, nk, 2, 1, dim, 16, 3, "none", kind)
        out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)), block_k=16)
        want, tol = ref.attention(*(ref.wide(t) for t in (q, k, v)), index, 16, None, dim ** -0.5, kind)
        close(out.numpy(), want, tol)


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_a_full_card_repeats_itself(mbx, ctx, kind, dim):
    """Several waves of CTAs, two an SM, give the same bits every time."""
    rng = np.random.default_rng(67)
    q, k, v = (up(ctx, ref.narrow(rng.standard_normal((2, 4096, h, dim)), kind)) for h in (16, 8, 8))
    index = mbx.block_select(q, k, 16, block_k=32)
    first = mbx.block_attention(q, k, v, index, block_k=32).numpy().tobytes()
    for _ in range(5):
        assert mbx.block_select(q, k, 16, block_k=32).numpy().tobytes() == index.numpy().tobytes()
        assert mbx.block_attention(q, k, v, index, block_k=32).numpy().tobytes() == first


@pytest.mark.skipif(importlib.util.find_spec("torch") is None, reason="captures with torch")
def test_a_captured_layer(mbx):
    """Heads, choice and attention in one graph, replayed on new inputs."""
    import torch
    rng = np.random.default_rng(71)
    n, tokens, heads, kv, dim = 2, 300, 4, 2, 40
    with mbx.Context(0) as ctx:
        x = ctx.empty((n, tokens, (heads + 2 * kv) * dim))
        pos = rng.integers(0, 30, (tokens, 3)).astype(np.float32)
        at = up(ctx, pos)
        parts = tuple(ctx.empty((n, tokens, h, dim), np.float16) for h in (heads, kv, kv))
        index, out = ctx.empty((n, heads, 3, 5), np.int32), ctx.empty(parts[0].shape)
        ws = mbx.block_select_workspace(parts[0], parts[1], 32), mbx.block_attention_workspace(parts[0], parts[1], index, 32)

        def call():
            mbx.qkv_norm_rope(x, heads, kv, dim, positions=at, axis_dims=(0, 20, 20), pairing="halves", out=parts)
            mbx.block_select(parts[0], parts[1], 5, block_k=32, workspace=ws[0], out=index)
            mbx.block_attention(*parts, index, block_k=32, workspace=ws[1], out=out)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        ctx.synchronize()
        ctx.set_stream(stream.cuda_stream)
        call()
        ctx.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for _ in range(2):
            host = rng.standard_normal(x.shape).astype(np.float32)
            mbx.check(mbx.abi.lib().mbx_memcpy_h2d(ctx.handle, x.vp, host.ctypes.data_as(ctypes.c_void_p), host.nbytes))
            ctx.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            wide = host.astype(np.float64).reshape(n, tokens, -1, dim)
            for got, part in zip(parts, (wide[:, :, :heads], wide[:, :, heads:heads + kv])):
                y, size = ref.norm_rope(part, None, 1e-6, True, pos[None], (0, 20, 20), 10000.0, True)
                close(got.numpy(), y, rope_tolerance(y, size, "f16"))
            q, k, v = (ref.wide(t.numpy()) for t in parts)
            assert np.array_equal(index.numpy(), ref.select(q, k, 5, 32))
            want, tol = ref.attention(q, k, v, index.numpy(), 32, None, dim ** -0.5, "f16")
            close(out.numpy(), want, tol)
        ctx.set_stream(None)
        del graph


@pytest.mark.parametrize("heads", [2, 148])
@pytest.mark.parametrize("nq", [2, 140])
@pytest.mark.parametrize("kind", DTYPES)
def test_block_attention_of_logits_beyond_a_step_of_one(mbx, ctx, kind, nq, heads):
    """Logits of up to 2^31, where f32 numbers are far more than one apart, and all of them exact: the largest takes all."""
    nk, dim = 640, 40
    rng = np.random.default_rng(73)
    steps = (np.arange(nk) * 37 % nk - 200) * (1 if kind == "bf16" else 64)  # distinct, 8 bits of bf16 at the top below
    if kind == "bf16":
        steps = np.where(np.abs(steps) > 255, -3, steps)
        steps[5] = 256
    q, k = np.zeros((1, nq, heads, dim)), np.zeros((1, nk, 1, dim))
    q[..., 0] = 2.0 ** (15 if kind == "f16" else 20) * np.where(np.arange(nq) % 2, 1, 0.75)[None, :, None]
    k[0, :, 0, 0] = steps
    size = 2.0 ** rng.integers(-6, 7, nk // 16).repeat(16)  # f32: another scale every 16 keys
    v = rng.standard_normal((1, nk, 1, dim)) * size[None, :, None, None]
    q, k, v = (ref.narrow(t, kind) for t in (q, k, v))
    index = np.broadcast_to(np.arange(10, dtype=np.int32), (1, heads, -(-nq // 128), 10)).copy()
    wide = ref.wide(v)[0, :, 0]
    for scale, best in ((1.0, steps.argmax()), (-1.0, steps.argmin())):
        if (steps == steps[best]).sum() > 1:
            continue
        out = mbx.block_attention(*(up(ctx, t) for t in (q, k, v, index)), scale=scale)
        want = np.broadcast_to(wide[best], q.shape)
        close(out.numpy(), want, 2.0 ** -20 * np.abs(want) + ref.HALF_STEP[kind] * np.abs(want))
