"""The operators of a drafted step at the ends of what they accept: lengths, bounds and numbers that an ordinary step does not bring.

As in tests/test_drafted_step_kernels_gpu.py, the same tests run without a GPU, between guard pages, when the environment says
RI_TEST_KERNELS=emulated; tests/test_drafted_step_ends.py starts that run."""
import numpy as np
import pytest
import torch

from test_drafted_step_kernels_gpu import (BF16_STEP, EMULATED, F32_STEP, PAGE, SharedCase, _guarded_buffers_go_back, drafted, f64, guarded, i32,  # noqa: F401
                                           int4_inputs, ops, plain_int4, pytestmark, softmax, starts, verify)


# ---------------------------------------------------------------- products with a matrix in 4 bits
@pytest.mark.parametrize("group", [512, 1024, 2 ** 30, 2 ** 31 - 128, 2 ** 31, 2 ** 32 + 128, 2 ** 40])
def test_products_in_4_bits_take_a_group_longer_than_the_matrix_as_one(ops, group):
    """One scale and zero point a row, whatever the group's length; whole numbers, so the sums are exact."""
    x, code, packed, scales, zero = int4_inputs(3, 20, 512, 512, True, torch.bfloat16, True, 3)
    xd, w, _, _ = plain_int4(x, code, scales, zero, 512)
    got = ops.gemm_int4_bf16(guarded(x), guarded(packed), guarded(scales), group, guarded(zero), torch.float32)
    assert np.array_equal(f64(got), xd @ w.T)


def test_the_c_entry_counts_groups_in_its_own_range(ops):
    """The largest group that its argument holds, straight to the C entry."""
    x, code, packed, scales, zero = int4_inputs(3, 20, 512, 512, True, torch.bfloat16, True, 4)
    xd, w, _, _ = plain_int4(x, code, scales, zero, 512)
    x, packed, scales, zero, out = guarded(x), guarded(packed), guarded(scales), guarded(zero), guarded(torch.zeros(3, 20))
    ops._call("ri_gemm_int4_bf16", out.data_ptr(), 0, x.data_ptr(), packed.data_ptr(), scales.data_ptr(), 1, zero.data_ptr(), 3, 20, 512,
              2 ** 31 - 128, ops._stream())
    assert np.array_equal(f64(out), xd @ w.T)


@pytest.mark.skipif(not EMULATED, reason="gigabytes that only the CPU's lazy memory gives for nothing")
@pytest.mark.parametrize("rows, n, k", [(1, 1, 2 ** 32 + 128), (1, 2 ** 32 + 16, 8)])
def test_products_in_4_bits_refuse_sizes_beyond_32_bits(ops, rows, n, k):
    """Each size's low 32 bits are those of a small product, which is not the one that was asked for."""
    from rust_inference_amd.errors import ShapeError
    group = -(-k // 128) * 128
    codes, scales = torch.empty(n, k // 2, dtype=torch.uint8), torch.empty(n, 1, dtype=torch.bfloat16)
    with pytest.raises(ShapeError):
        ops.gemm_int4_bf16(torch.empty(rows, k, dtype=torch.bfloat16), codes, scales, group)


FORMS = [  # rows, n, k, group: the forms of a whole machine and, on one of one compute unit, the one that holds x
    (1, 16, 128, 128), (3, 40, 1160, 64), (17, 48, 264, 32), (45, 50, 200, 64), (65, 18, 416, 32), (16, 200, 2080, 64), (9, 331, 4096, 128),
    (2, 100, 1408, 384), (130, 16, 128, 64),
]
if not EMULATED:
    FORMS += [(16, 9001, 1056, 64), (8, 16500, 2048, 32), (5, 8210, 4096, 256), (40, 8300, 200, 64), (20, 8200, 640, 128), (49, 33001, 136, 64)]


@pytest.mark.parametrize("rows, n, k, group", FORMS)
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("exponent", [100, 112, 125, -60, -100])
def test_products_in_4_bits_of_very_large_and_very_small_x_are_exact(ops, rows, n, k, group, zeros, exponent):
    """Whole numbers up to 4 times a power of two, scales of such a power that results stay in range: the same exact products, shifted.  (The
    largest x, 2^127; the smallest sums are multiples of 2^-3 x 2^-100 x 2^-12, a normal number.)"""
    x, code, packed, scales, zero = int4_inputs(rows, n, k, group, zeros, torch.float32, True, 5)
    down = 40 if exponent > 0 else 0
    want = np.ldexp(x.double().numpy() @ plain_int4(x, code, scales, zero, group)[1].T, exponent - down)
    assert np.abs(want).max() < 2.0 ** 127
    got = ops.gemm_int4_bf16(guarded(torch.ldexp(x.float(), torch.tensor(exponent)).to(torch.bfloat16)), guarded(packed),
                             guarded(torch.ldexp(scales, torch.tensor(-down))), group, guarded(zero), torch.float32)
    assert np.array_equal(f64(got), want)


@pytest.mark.parametrize("rows, n, k, group", FORMS)
@pytest.mark.parametrize("scale", [2.0 ** -12, 2.0 ** -30])
def test_products_in_4_bits_of_the_largest_numbers(ops, rows, n, k, group, scale):
    """Every x is the largest bfloat16 number, of one sign in the first row; up to K / 2^12 of float32's range goes into a sum of |scale x|.  Bounds
    as for ordinary x: an addition is off by half a step of a partial sum."""
    _, code, packed, _, zero = int4_inputs(rows, n, k, group, True, torch.float32, False, 6)
    g = torch.Generator().manual_seed(7)
    x = torch.full((rows, k), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16)
    x[1:] *= (torch.randint(0, 2, (rows - 1, k), generator=g) * 2 - 1).to(torch.bfloat16)
    scales = scale * (0.5 + 0.5 * torch.rand(n, -(-k // group), generator=g))
    xd, w, s, z = plain_int4(x, code, scales, zero, group)
    want, size = xd @ w.T, np.abs(xd) @ (s * (32.0 + code.double().numpy() + z)).T
    bound = F32_STEP * (128 + 4 + -(-k // 128) + 8) * size
    got = f64(ops.gemm_int4_bf16(guarded(x), guarded(packed), guarded(scales), group, guarded(zero), torch.float32))
    fits = np.abs(want) + bound < np.finfo(np.float32).max
    assert fits[1:].all() and fits.any(0).all() if scale < 2.0 ** -20 else fits.any()
    assert (np.abs(got - want)[fits] <= bound[fits]).all()
    assert np.isinf(got[np.abs(want) - bound > np.finfo(np.float32).max]).all()


@pytest.mark.parametrize("rows, n, k, group", FORMS)
def test_products_in_4_bits_at_the_small_end(ops, rows, n, k, group):
    """x of some 2^-118: results are off by what ordinary ones are and, an operation, 2^12 times half the least step of float32 (2^-149), times the
    scale below 1 where it is not the last one."""
    x, code, packed, scales, zero = int4_inputs(rows, n, k, group, True, torch.float32, False, 8)
    x = torch.ldexp(x.float(), torch.tensor(-118)).to(torch.bfloat16)
    xd, w, s, z = plain_int4(x, code, scales, zero, group)
    count = 128 + 4 + -(-k // 128) + 8
    bound = F32_STEP * count * (np.abs(xd) @ (s * (32.0 + code.double().numpy() + z)).T) + 2.0 ** -138 * (k + count)
    got = f64(ops.gemm_int4_bf16(guarded(x), guarded(packed), guarded(scales), group, guarded(zero), torch.float32))
    assert (np.abs(got - xd @ w.T) <= bound).all()


def off_its_start(t, by):
    """The same numbers behind ``by`` others of a larger tensor."""
    whole = torch.zeros(t.numel() + by, dtype=t.dtype)
    whole[by:] = t.reshape(-1)
    return guarded(whole)[by:].view(t.shape)


@pytest.mark.parametrize("rows, n, k, group", FORMS)
def test_products_in_4_bits_of_operands_that_start_anywhere(ops, rows, n, k, group):
    """Codes on a 4-byte boundary and no larger one, scales and zero points on one of their own size: the same bits."""
    x, _, packed, scales, zero = int4_inputs(rows, n, k, group, True, torch.bfloat16, False, 9)
    want = ops.gemm_int4_bf16(guarded(x), guarded(packed), guarded(scales), group, guarded(zero), torch.float32)
    got = ops.gemm_int4_bf16(guarded(x), off_its_start(packed, 4), off_its_start(scales, 1), group, off_its_start(zero, 3), torch.float32)
    assert torch.equal(got, want)


# ---------------------------------------------------------------- attention over pages that the batch shares
@pytest.mark.parametrize("change", [dict(max_len=2 ** 32 + 100), dict(max_len=2 ** 40), dict(shared=2 ** 37 + 64), dict(shared=2 ** 40)])
def test_attention_over_shared_pages_refuses_lengths_that_no_table_holds(ops, change):
    """Among them such whose low 32 bits, or whose pages' low 32 bits, are those of the case."""
    from rust_inference_amd.errors import ShapeError
    c = SharedCase([(1, 36)], 64, 4, 2, 64)
    with pytest.raises(ShapeError):
        c.run(ops, **change)


def test_attention_over_shared_pages_allocates_nothing_for_a_length_that_it_refuses(ops, monkeypatch):
    from rust_inference_amd.errors import ShapeError
    c = SharedCase([(1, 36)], 64, 4, 2, 64)
    class Torch:
        def __getattr__(self, name):
            assert name != "empty"
            return getattr(torch, name)
    args = dict(k=guarded(c.k), v=guarded(c.v), qkv=guarded(c.qkv))
    monkeypatch.setattr(ops, "torch", Torch())
    for max_len in (0, -1, 32 * c.width + 1, 2 ** 31 - 1):
        with pytest.raises(ShapeError):
            c.run(ops, max_len=max_len, **args)


def test_attention_over_shared_pages_takes_any_bound_of_the_new_tokens(ops):
    """Far above the tokens that there are, its low 32 bits 0 or small."""
    c = SharedCase([(3, 40), (1, 9)], 64, 4, 2, 64, seed=2)
    for c.max_new in (3, 100, 2 ** 31 - 1, 2 ** 32, 2 ** 32 + 1):
        c.check(c.run(ops))


def test_attention_over_shared_pages_refuses_lengths_whose_chunks_pass_32_bits(ops):
    """The widest tables, and lengths within a chunk of 2^31: the count of own chunks is taken in 64 bits, and refused."""
    from rust_inference_amd.errors import KernelError
    c = SharedCase([(1, 36)], 64, 4, 2, 64)
    for width, max_len in ((2 ** 26 - 1, 2 ** 31 - 40), (2 ** 26 - 1, 2 ** 31 - 200), (2 ** 26 - 17, 2 ** 31 - 16 * 32 - 40)):
        c.table = torch.zeros(1, width, dtype=torch.int32)
        with pytest.raises(KernelError):
            c.run(ops, max_len=max_len)
    # (chunks of eight pages or, on a machine with fewer compute units than the sequence has key heads, sixteen)
    assert ops._get("ri_attention_shared_slots")(1, 1, 1, 0, 2 ** 31 - 1, 4, 2) in (2 ** 22, 2 ** 23)
    assert ops._get("ri_attention_shared_slots")(1, 1, 1, 2 ** 27, 100, 4, 2) > 0


@pytest.mark.parametrize("lens, shared, heads, kv, dim", [([(20, 40), (1, 30)], 64, 4, 2, 64), ([(9, 700), (3, 3), (30, 33)], 32, 8, 1, 32),
                                                          ([(17, 18)], 0, 16, 4, 128), ([(6, 6), (0, 0), (40, 600)], 320, 2, 2, 128)])
def test_attention_over_shared_pages_answers_sequences_that_bring_more_than_the_bound(ops, lens, shared, heads, kv, dim):
    """max_new sizes the grid; a sequence above it takes longer and gets what it asked for."""
    c = SharedCase(lens, shared, heads, kv, dim, seed=11)
    for c.max_new in (1, 4, c.max_new):
        c.check(c.run(ops))


@pytest.mark.parametrize("heads, kv, dim", [(4, 2, 64), (16, 1, 32), (8, 2, 128)])
def test_attention_over_shared_pages_takes_a_sequences_tokens_in_any_order(ops, heads, kv, dim):
    """The positions of a sequence fall, repeat or jump; every token sees the keys up to its own, chunks beyond the last token's among them."""
    c = SharedCase([(3, 1400), (1, 30), (70, 600), (5, 300)], 64, heads, kv, dim, seed=12)
    rng = np.random.default_rng(12)
    c.pos[:3] = [64 + 1399, 64 + 2, 64 + 700]
    c.pos[4:74] = (64 + rng.permutation(np.r_[599, rng.integers(0, 599, 69)])).tolist()
    c.pos[74:] = [64 + 299, 64 + 299, 10, 64, 63]
    q, k, v = c.qkv[:, :heads * dim].double().view(-1, heads, dim).numpy(), c.k.double(), c.v.double()
    got, per, seq = f64(c.run(ops)), heads // kv, np.repeat(np.arange(4), c.counts)
    assert np.isfinite(got).all()
    for t, p in enumerate(c.pos):
        pages = c.table[seq[t], :p // PAGE + 1].long()
        for h in range(heads):
            keys = k[pages, h // per].reshape(-1, dim)[:p + 1].numpy()
            values = v[pages, h // per].transpose(1, 2).reshape(-1, dim)[:p + 1].numpy()
            s = keys @ q[t, h] * c.scale
            w = np.exp(s - s.max())
            w /= w.sum()
            want, size = w @ values, w @ np.abs(values)
            # (the weights and the result rounded to bfloat16 once each; float32 scores, as SharedCase.check derives)
            assert (np.abs(got[t, h * dim:(h + 1) * dim] - want) <= BF16_STEP * np.abs(want) + (BF16_STEP + 2.0 ** -14) * size).all(), (t, h)


@pytest.mark.parametrize("heads, kv, dim", [(4, 2, 64), (16, 1, 32), (40, 2, 128)])
@pytest.mark.parametrize("max_len", [1, 31, 33, 160, 161, 192, 193, 350, 900, 1161])
def test_attention_over_shared_pages_sees_no_key_behind_the_bound(ops, heads, kv, dim, max_len):
    """What lies at max_len and behind it, shared or own, within a page, a chunk or a run, is as if a token's position came before it."""
    c = SharedCase([(1, 1000), (3, 40), (2, 600)], 160, heads, kv, dim, seed=13)
    got = c.run(ops, max_len=max_len)
    c.pos = [min(p, max_len - 1) for p in c.pos]
    c.check(got)


def test_attention_over_shared_pages_refuses_a_scale_that_its_exponents_do_not_hold(ops):
    """Scores are taken times log2(e)."""
    from rust_inference_amd.errors import KernelError
    c = SharedCase([(1, 36)], 64, 4, 2, 64)
    for c.scale in (3e38, 2.4e38, float("nan"), -1.0):
        with pytest.raises(KernelError):
            c.run(ops)


@pytest.mark.parametrize("heads", [4, 40])
def test_attention_over_shared_pages_of_scores_up_to_a_billion(ops, heads):
    """Whole queries and keys up to 8: dot products are exact and at most 4,096, times 2^17 the scores reach 5e8.  The largest score's
    product with log2(e), below 2^30, is off by at most 2^5, which is the exponent that all weights of a column share."""
    c = SharedCase([(1, 36), (3, 70)], 192, heads, 2, 64, seed=14)
    whole = lambda t: torch.where(t.isnan(), t, torch.randint(-8, 9, t.shape, generator=torch.Generator().manual_seed(15)).to(t.dtype))  # noqa: E731
    c.k, c.qkv, c.scale = whole(c.k), whole(c.qkv), 2.0 ** 17
    c.check(c.run(ops))


@pytest.mark.parametrize("heads", [4, 40])
def test_attention_over_shared_pages_leaves_rows_before_the_sequences_at_zero(ops, heads):
    """Two rows of NaN before the first sequence and one behind the last, which are no sequence's; the others as without them."""
    c = SharedCase([(2, 10), (1, 35), (3, 300)], 96, heads, 2, 64, seed=18)
    want = c.run(ops)
    c.check(want)
    pad = torch.full((2, c.qkv.shape[1]), float("nan"), dtype=torch.bfloat16)
    c.qkv, c.pos = torch.cat([pad, c.qkv, pad[:1]]), [3, 10 ** 9] + c.pos + [-2]
    got = ops.attention_shared_bf16(guarded(c.qkv), guarded(c.k), guarded(c.v), i32(2 + starts(c.counts)), i32(c.pos), guarded(c.table), 3, c.max_new,
                                    c.shared, c.max_len, heads, 2, 64, c.scale)
    assert (f64(got)[[0, 1, 8]] == 0).all() and torch.equal(got[2:8], want)


@pytest.mark.parametrize("which", ["k", "v", "qkv"])
def test_attention_over_shared_pages_refuses_what_does_not_start_on_16_bytes(ops, which):
    from rust_inference_amd.errors import KernelError
    c = SharedCase([(1, 36)], 64, 4, 2, 64)
    t = getattr(c, which)
    off = guarded(torch.zeros(t.numel() + 8, dtype=torch.bfloat16))[1:1 + t.numel()].view(t.shape)
    with pytest.raises(KernelError):
        c.run(ops, **{which: off})


# ---------------------------------------------------------------- drafted tokens
@pytest.mark.skipif(not EMULATED, reason="gigabytes that only the CPU's lazy memory gives for nothing")
@pytest.mark.parametrize("rows, vocab", [(1, 2 ** 32 + 40), (2 ** 32 + 1, 1)])
def test_drafts_with_sizes_beyond_32_bits_are_refused(ops, rows, vocab):
    from rust_inference_amd.errors import ShapeError
    logits, tokens = torch.empty(rows, vocab), torch.empty(rows, dtype=torch.int32)
    with pytest.raises(ShapeError):
        ops.verify_drafts(logits, tokens, i32([0, 1]), None, 0.0)


@pytest.mark.parametrize("vocab", [1, 3, 300, 4096, 9000])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_a_row_that_masks_everything_lets_no_draft_stand(ops, vocab, temperature):
    """Token 0 among the drafts, which is also the token that such a row gives; a row before it in which 0 is the best lets it stand."""
    masked = np.full((5, vocab), -np.inf, dtype=np.float32)
    masked[1::2] = np.nan
    u = np.zeros(5)
    accepted, out = verify(ops, masked, None, np.array([0, 0, 0, 0, 0]), [2, 3], u, temperature)
    assert accepted.tolist() == [0, 0] and out.tolist() == [0, -1, 0, -1, -1]
    masked[2, 0] = masked[0, vocab - 1] = -3e38
    accepted, out = verify(ops, masked, None, np.array([0, vocab - 1, 0, 0, 0]), [2, 3], u, temperature)
    assert accepted.tolist() == [1, 1] and out.tolist() == [vocab - 1, 0, 0, 0, -1]


@pytest.mark.parametrize("vocab", [10, 4096, 9001])
def test_greedy_takes_an_infinity_for_the_largest_number(ops, vocab):
    """The first of an infinity and the largest finite number is the best, whichever of them it is, in one chunk or in two; with a
    temperature both weigh one half."""
    top = np.finfo(np.float32).max
    logits = np.zeros((4, vocab), dtype=np.float32)
    first, second = 3, vocab - 1
    logits[0, [first, second]], logits[1, [first, second]], logits[2, [first, second]] = (top, np.inf), (np.inf, top), (np.inf, np.inf)
    logits[3, [first, second]], logits[:, 1], logits[:, 2] = (np.nextafter(top, np.float32(0)), np.inf), np.nan, -np.inf
    tokens = np.array([0, first, first, first])
    accepted, out = verify(ops, logits, None, tokens, [4], None, 0.0)
    assert accepted.tolist() == [3] and out.tolist() == [first, first, first, second]
    accepted, out = verify(ops, logits[:2], None, tokens[:2], [2], np.array([0.25, 0.75]), 1.0)
    assert accepted.tolist() == [1] and out.tolist() == [first, second]


@pytest.mark.parametrize("vocab", [7, 4097, 9000])
def test_greedy_takes_no_nan_for_a_number(ops, vocab):
    """NaN at the lowest ids, at every other one and everywhere but one."""
    logits = np.full((3, vocab), np.nan, dtype=np.float32)
    logits[0, 2:], logits[1, 1::2], logits[2, vocab - 2] = -5.0, -np.inf, -3e38
    logits[0, 5] = 1.0
    accepted, out = verify(ops, logits, None, np.array([0, 5, 0]), [3], None, 0.0)
    assert accepted.tolist() == [1] and out.tolist() == [5, 0, -1]
    accepted, out = verify(ops, logits[2:], None, np.array([0]), [1], None, 0.0)
    assert accepted.tolist() == [0] and out.tolist() == [vocab - 2]


@pytest.mark.parametrize("temperature", [1e-20, 1e-24, 1.1e-24, 1.3e-24, 1e-30, 1e-36, 1e-40, 1e-44, 1e-46, 3e-47, 1e-47, 1e-48, 1e-60, 1e-200, 1e-300, 5e-324])
@pytest.mark.parametrize("top", [0.0, 1e-38, -1e-38, 1.5, -40.0])
def test_the_coldest_temperatures(ops, temperature, top):
    """A largest logit of 0, as where logits are shifted to it, or a small, an ordinary one; entries 2^-149, the least that float32 tells apart,
    to 2^-126 below it.  Every entry weighs 0, the same as the largest or, at temperatures about that distance, something in between."""
    vocab, counts = 4200, [3, 3, 2]
    rng = np.random.default_rng(16)
    logits = (top - 0.1 - np.abs(rng.standard_normal((8, vocab)))).astype(np.float32)
    best = rng.integers(0, vocab, 8)
    logits[np.arange(8), best] = top
    for r, d in enumerate((1e-45, 3e-45, 1e-43, 1e-40, 1.2e-38, 1e-37, 1e-35, 1e-30)):
        logits[r, (best[r] + 7) % vocab] = np.float32(np.float64(np.float32(top)) - d)
    logits[:, 11][best != 11] = -np.inf
    tokens = np.roll(best, 1)
    tokens[4] = (best[3] + 7) % vocab                        # the entry a little below the best
    u = np.full(8, 0.3, dtype=np.float32)
    near = (logits.astype(np.float64) - logits.max(1, keepdims=True).astype(np.float64))
    with np.errstate(over="ignore"):
        p = np.exp(near / temperature)
    p /= p.sum(1, keepdims=True)
    accepted, out, at = [], [], 0
    for n in counts:                                          # looked-up drafts: a draft stands if u < p, else it is taken out
        stop = next((r for r in range(at, at + n - 1) if not u[r] < p[r, tokens[r + 1]]), at + n - 1)
        weights = p[stop].copy()
        if stop < at + n - 1:
            weights[tokens[stop + 1]] = 0.0
            if not weights.sum() > 0:
                weights = p[stop]
        upto = np.cumsum(weights)
        target = float(u[at + n - 1]) * upto[-1]
        # (nothing lies within 1e-9 of a border, far above what an exponential and a sum of two such entries are off by)
        assert np.abs(upto[weights > 0] - target).min() > 1e-9 * upto[-1] and all(abs(p[r, tokens[r + 1]] - u[r]) > 1e-9 for r in range(at, at + n - 1))
        accepted.append(stop - at)
        out += tokens[at + 1:stop + 1].tolist() + [int((upto > target).argmax())] + [-1] * (at + n - 1 - stop)
        at += n
    got = verify(ops, logits, None, tokens, counts, u, temperature)
    assert got[0].tolist() == accepted and got[1].tolist() == out
    # drafts drawn from the target itself: q = p, and every one that has any weight stands
    got = verify(ops, logits, np.roll(logits, 1, 0), np.roll(best, 1), counts, u, temperature)
    assert got[0].tolist() == [n - 1 for n in counts]


@pytest.mark.skipif(not EMULATED, reason="a row that must not be read lies in a guard page")
@pytest.mark.parametrize("vocab", [40, 4097])
def test_draft_logits_of_tokens_that_are_no_drafts_are_not_read(ops, vocab):
    """The C entry is told of a row before the buffer's first, which is that of a sequence's first token."""
    import emulated
    logits, draft, tokens, u = drafted([3], vocab, 1.0, True, 17)
    held = emulated.tensor(torch.tensor(draft[1:]), "draft logits", flush_end=False)
    t = lambda a: guarded(torch.tensor(np.ascontiguousarray(a), dtype=torch.float32))  # noqa: E731
    args, cu, ids = (t(logits), t(u)), i32([0, 3]), i32(tokens)
    words = ops._get("ri_verify_drafts_workspace_words")(1, 3, vocab, 1)
    accepted, out, ws = i32([0]), i32([0, 0, 0]), guarded(torch.zeros(words, dtype=torch.float64))
    ops._call("ri_verify_drafts", accepted.data_ptr(), out.data_ptr(), args[0].data_ptr(), held.data_ptr() - 4 * vocab, ids.data_ptr(), cu.data_ptr(),
              args[1].data_ptr(), ws.data_ptr(), 1, 3, vocab, 1.0, 0)
    want = verify(ops, logits, draft, tokens, [3], u, 1.0)
    assert np.array_equal(accepted.numpy(), want[0]) and np.array_equal(out.numpy(), want[1])


@pytest.mark.parametrize("p_row, q_row, temperature", [([1.0, 0.2, -1.5], [-1.2, 0.8, 0.5], 1.0)] if EMULATED else
                         [([1.0, 0.2, -1.5], [-1.2, 0.8, 0.5], 1.0), ([0.5, -2.0, 1.0, 0.3, 2.5], [2.0, 1.0, 0.5, -1.0, 0.0], 0.7),
                          ([3.0, 0.0, 0.0, 0.0, -1.0, 1.0], [0.0, 0.0, 1.0, 2.0, 0.0, 0.0], 1.5)])
def test_the_first_token_put_out_has_the_targets_probabilities(ops, p_row, q_row, temperature):
    """Every pair of numbers of a grid and every draft, weighed by the draft's distribution.  Of g midpoints as many lie below a border as its
    place times g, give or take one half.  So a draft's share of acceptances is off by 1 / 2g at most, a token's share of the draws from what
    is left, between two borders, by 1 / g, and the token t's probability by (q_t + r_t) / 2g + (1 - acceptance) / g, with r what is left, made a
    distribution.  Neither drawing from p after a fall nor letting every draft stand would keep within that."""
    vocab, grid = len(p_row), 16 if EMULATED else 64
    p_row, q_row = np.array(p_row, dtype=np.float32), np.array(q_row, dtype=np.float32)
    p, q = softmax(p_row, temperature), softmax(q_row, temperature)
    left = np.maximum(p - q, 0.0)
    fallen, left = left.sum(), left / left.sum()
    bound = (q + left) / (2 * grid) + fallen / grid + 1e-9
    for wrong in (np.minimum(p, q) + fallen * p, q, p[::-1]):
        assert (np.abs(wrong - p) > 2 * bound).any()
    cells = [(d, a, b) for d in range(vocab) for a in range(grid) for b in range(grid)]
    tokens = np.array([[0, d] for d, _, _ in cells]).reshape(-1)
    u = np.array([[(a + 0.5) / grid, (b + 0.5) / grid] for _, a, b in cells]).reshape(-1)
    _, out = verify(ops, np.tile(p_row, (2 * len(cells), 1)), np.tile(q_row, (2 * len(cells), 1)), tokens, [2] * len(cells), u, temperature)
    found = np.bincount(out[::2], weights=np.repeat(q, grid * grid) / grid ** 2, minlength=vocab)
    assert (np.abs(found - p) <= bound).all(), (found, p, bound)


@pytest.mark.parametrize("vocab", [4100, 9000])
@pytest.mark.parametrize("temperature", [0.8, 0.0])
def test_drafts_are_verified_from_logits_that_start_anywhere(ops, vocab, temperature):
    """On a 4-byte boundary and no larger one."""
    counts = [3, 1, 4]
    logits, draft, tokens, u = drafted(counts, vocab, 0.8, True, 19)
    want = verify(ops, logits, draft, tokens, counts, u, temperature)
    for by in ((1, 0), (0, 1), (3, 2)):
        t = [off_its_start(torch.tensor(a), o) for a, o in zip((logits, draft), by)]
        got = ops.verify_drafts(t[0], i32(tokens), i32(starts(counts)), off_its_start(torch.tensor(u), 1), temperature, t[1])
        assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])


# ---------------------------------------------------------------- streams and graphs
def step_inputs(seed, new, own):
    """The device operands of a step: attention of ``new`` tokens a sequence behind 128 shared ones, a product, a verification."""
    c = SharedCase([(n, m) for n, m in zip(new, own)], 128, 8, 2, 64, seed=seed, table_spare=24 - -(-max(own) // PAGE))
    x, _, packed, scales, zero = int4_inputs(6, 40, 512, 64, True, torch.bfloat16, False, seed)
    logits, draft, tokens, u = drafted(new, 5000, 1.0, True, seed)
    f = lambda a: torch.tensor(a, dtype=torch.float32, device="cuda:0")  # noqa: E731
    return [t.to("cuda:0") for t in (c.qkv, c.table, x, packed, scales, zero)] + [f(logits), f(draft), f(u), i32(tokens), i32(c.pos),
                                                                                  i32(starts(new))], (c.k.to("cuda:0"), c.v.to("cuda:0"))


def step_calls(ops, a, pages, max_new, max_len):
    qkv, table, x, packed, scales, zero, logits, draft, u, tokens, pos, cu = a
    return [ops.attention_shared_bf16(qkv, *pages, cu, pos, table, 3, max_new, 128, max_len, 8, 2, 64, 0.125),
            ops.gemm_int4_bf16(x, packed, scales, 64, zero), *ops.verify_drafts(logits, tokens, cu, u, 0.8, draft),
            *ops.verify_drafts(logits, tokens, cu, None, 0.0)]


@pytest.mark.skipif(EMULATED, reason="streams")
def test_two_steps_at_once_on_two_streams(ops):
    """Neither waits for the other; each gives what it gives alone."""
    cases = [step_inputs(41, [2, 1, 3], [40, 600, 3]), step_inputs(42, [1, 4, 1], [500, 90, 33])]
    want = [[t.clone() for t in step_calls(ops, a, p, 4, 128 + 700)] for a, p in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for i, (a, p) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(step_calls(ops, a, p, 4, 128 + 700))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, w) for step in got[i] for g, w in zip(step, want[i]))


@pytest.mark.skipif(EMULATED, reason="graphs")
def test_a_captured_step_answers_other_lengths_positions_and_counts(ops):
    """One graph, captured for two tokens a sequence, replayed over steps whose sequences bring others in number, more than two among them, at
    other positions: every replay gives the eager bits of a call with the same bounds."""
    pages = None
    steps = []
    for seed, new, own in ((51, [2, 2, 2], [40, 600, 3]), (52, [1, 4, 1], [500, 90, 33]), (53, [6, 0, 0], [700, 1, 1]), (54, [0, 1, 5], [2, 1, 321])):
        a, pages = step_inputs(seed, new, own)
        steps.append((a, pages))
    most = max(p[0].shape[0] for _, p in steps)
    held_pages = [torch.zeros((most, *t.shape[1:]), dtype=t.dtype, device=t.device) for t in pages]
    held = [t.clone() for t in steps[0][0]]
    def put(a, p):
        for h, t in zip(held, a):
            h.copy_(t)
        for h, t in zip(held_pages, p):
            h[:t.shape[0]].copy_(t)
    eager = []
    for a, p in steps:
        put(a, p)
        eager.append([t.clone() for t in step_calls(ops, held, held_pages, 2, 128 + 700)])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step_calls(ops, held, held_pages, 2, 128 + 700)
    for turn in range(9):
        i = turn * 3 % 4
        put(*steps[i])
        graph.replay()
        torch.ones(1000, device="cuda:0").sum()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(out, eager[i])), (turn, i)
