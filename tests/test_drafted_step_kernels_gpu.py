"""The operators of a drafted step alone against plain ones in 64 bits: products with a matrix in 4 bits, attention over pages
that the batch shares, drafted tokens held to the target's distribution.

The same tests run without a GPU when the environment says RI_TEST_KERNELS=emulated (tests/emulated.py): then every operand lies
between guard pages.  tests/test_drafted_step.py starts that run."""
import os

import numpy as np
import pytest
import torch

EMULATED = os.environ.get("RI_TEST_KERNELS") == "emulated"
pytestmark = [] if EMULATED else pytest.mark.gpu
DEV = "cpu" if EMULATED else "cuda:0"
BF16_STEP = 2.0 ** -8                    # what one rounding to bfloat16 is off by at most, relative to the value
F32_STEP = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    if EMULATED:
        import emulated
        return emulated.ops()
    from rust_inference_amd.kernels import ops
    return ops


@pytest.fixture(autouse=True)
def _guarded_buffers_go_back():
    yield
    if EMULATED:
        import gc
        import emulated
        gc.collect()
        emulated.free_all()


def guarded(x):
    if x is None:
        return None
    if EMULATED:
        import emulated
        return emulated.tensor(x.contiguous(), "a test's operand")
    return x.to(DEV)


def i32(a):
    return guarded(torch.tensor(np.asarray(a), dtype=torch.int32))


def f64(x):
    return x.detach().to("cpu", torch.float64).numpy()


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


# ---------------------------------------------------------------- products with a matrix in 4 bits
def int4_inputs(rows, n, k, group, zeros, scale_type, whole, seed=0):
    """x, codes, scales and zero points on the CPU; ``whole``: small whole numbers and powers of two, whose products and sums are
    exact in float32."""
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    code = torch.randint(0, 16, (n, k), generator=g)
    packed = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)
    if whole:
        x = torch.randint(-4, 5, (rows, k), generator=g).to(torch.bfloat16)
        scales = (2.0 ** torch.randint(-3, 3, (n, groups), generator=g)).to(scale_type)
    else:
        x = torch.randn(rows, k, generator=g).to(torch.bfloat16)
        scales = (0.02 * torch.randn(n, groups, generator=g)).to(scale_type)
    zero = torch.randint(0, 16, (n, groups), generator=g).to(torch.uint8) if zeros else None
    return x, code, packed, scales, zero


def plain_int4(x, code, scales, zero, group):
    k = code.shape[1]
    s = scales.double().repeat_interleave(group, 1)[:, :k]
    z = 8.0 if zero is None else zero.double().repeat_interleave(group, 1)[:, :k]
    return x.double().numpy(), ((code.double() - z) * s).numpy(), s.abs().numpy(), np.broadcast_to(np.asarray(z, dtype=np.float64), code.shape)


INT4 = [  # rows, n, k, group, zeros
    (1, 16, 128, 128, False), (1, 1, 8, 32, True), (3, 17, 136, 64, True), (8, 40, 1024, 128, True), (16, 33, 512, 32, True),
    (17, 48, 264, 32, False), (31, 20, 384, 256, True), (45, 50, 200, 64, False), (64, 64, 256, 128, True), (65, 18, 160, 32, True),
    (130, 16, 128, 64, True), (2, 100, 1408, 384, False), (5, 35, 2568, 128, True),
    # (on a machine made small these go by the kernel that holds x: sixteen and more pieces of 128 columns, one tile and several a workgroup)
    (16, 200, 2080, 64, True), (9, 331, 4096, 128, False), (1, 200, 1056, 32, True), (13, 900, 2048, 256, True), (16, 500, 3968, 32, False),
]
if not EMULATED:                          # and on a whole one these do; the last by two, four and four times two tiles
    INT4 += [(3, 8300, 512, 128, True), (16, 9001, 1056, 64, False), (8, 16500, 2048, 32, True), (5, 8210, 4096, 256, True),
             (16, 50001, 264, 32, True), (2, 8300, 4352, 128, False), (40, 8300, 200, 64, True), (20, 8200, 640, 128, False),
             (45, 2560, 1032, 32, True), (49, 33001, 136, 64, True), (256, 4100, 512, 128, False), (129, 5000, 264, 32, True)]


@pytest.mark.parametrize("rows, n, k, group, zeros", INT4)
@pytest.mark.parametrize("scale_type", [torch.bfloat16, torch.float32])
def test_products_in_4_bits_of_whole_numbers_are_exact(ops, rows, n, k, group, zeros, scale_type):
    """|x| <= 4 and codes as 16 to 31: a group's sum of products is below 2^14 up to 128 columns, all sums are multiples of 2^-3 below
    2^20, so float32 holds every one of them and the result is the exact one."""
    x, code, packed, scales, zero = int4_inputs(rows, n, k, group, zeros, scale_type, True)
    got = ops.gemm_int4_bf16(guarded(x), guarded(packed), guarded(scales), group, guarded(zero), torch.float32)
    xd, w, _, _ = plain_int4(x, code, scales, zero, group)
    assert np.array_equal(f64(got), xd @ w.T)


@pytest.mark.parametrize("rows, n, k, group, zeros", INT4)
@pytest.mark.parametrize("out_type", [torch.bfloat16, torch.float32])
def test_products_in_4_bits(ops, rows, n, k, group, zeros, out_type):
    """Every addition on the way of an output rounds by half a step of a partial sum that the sum of |scale| |x| (16 + code) and of
    |scale| |x| (16 + zero) bounds; there are at most 128 of them in a piece of 128 columns for each sum, four for its scale and zero
    point and one a piece and wavefront; then one rounding of the result."""
    x, code, packed, scales, zero = int4_inputs(rows, n, k, group, zeros, torch.bfloat16, False, 1)
    got = f64(ops.gemm_int4_bf16(guarded(x), guarded(packed), guarded(scales), group, guarded(zero), out_type))
    xd, w, s, z = plain_int4(x, code, scales, zero, group)
    want = xd @ w.T
    size = np.abs(xd) @ (s * (32.0 + code.double().numpy() + z)).T
    bound = F32_STEP * (128 + 4 + -(-k // 128) + 8) * size
    if out_type == torch.bfloat16:
        bound = bound + BF16_STEP * np.abs(want) * (1 + 1e-3)
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()


def test_products_in_4_bits_find_one_weight(ops):
    """One column of x is not zero, and the matrix's entry there is what comes out: every code, at every place of a piece."""
    n, k = 16, 256
    code = torch.arange(n)[:, None].expand(n, k) + torch.arange(k)[None, :] & 15
    packed = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)
    scales = torch.ones(n, 8, dtype=torch.bfloat16)
    for at in range(0, k, 64):
        x = torch.zeros(64, k, dtype=torch.bfloat16)
        x[torch.arange(64), at + torch.arange(64)] = 1.0
        got = ops.gemm_int4_bf16(guarded(x), guarded(packed), guarded(scales), 32, None, torch.float32)
        assert np.array_equal(f64(got), (code[:, at:at + 64].t() - 8).double().numpy())


def test_products_in_4_bits_refuse_what_they_do_not_take(ops):
    from rust_inference_amd.errors import InferenceError, KernelError, ShapeError
    x, code, packed, scales, zero = int4_inputs(2, 16, 128, 32, True, torch.bfloat16, False)
    x, packed, scales, zero = guarded(x), guarded(packed), guarded(scales), guarded(zero)
    for group in (0, 16, 48, 96, 200, -128):
        with pytest.raises(ShapeError):
            ops.gemm_int4_bf16(x, packed, scales, group, zero)
    for bad in ((x.float(), packed, scales, zero), (x, packed[:, :60].contiguous(), scales, zero), (x, packed, scales[:, :3].contiguous(), zero),
                (x, packed, scales.half(), zero), (x, packed, scales, zero.to(torch.int8)), (x, packed, scales, zero[:8].contiguous()),
                (x[:0], packed, scales, zero), (x[:, :60].contiguous(), packed[:, :30].contiguous(), scales[:, :2].contiguous(), None),
                (x, packed.t(), scales, zero), (x[0], packed, scales, zero)):
        with pytest.raises(InferenceError):
            ops.gemm_int4_bf16(bad[0], bad[1], bad[2], 32, bad[3])
    with pytest.raises(ShapeError):
        ops.gemm_int4_bf16(x, packed, scales, 32, zero, torch.float16)
    whole = torch.zeros(16 * 64 + 8, dtype=torch.uint8, device=DEV)
    with pytest.raises(KernelError):                          # codes off a 4-byte boundary
        ops.gemm_int4_bf16(x, whole[1:1 + 16 * 64].view(16, 64), scales, 32, zero)


# ---------------------------------------------------------------- attention over pages that the batch shares
PAGE = 32


class SharedCase:
    """Sequences of (new tokens, tokens behind the shared ones with the new ones); what no key was written to holds NaN."""

    def __init__(self, lens, shared, heads, kv, dim, q_off=0, seed=0, spare=3, table_spare=2, pad_rows=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.shared, self.heads, self.kv, self.dim, self.q_off = lens, shared, heads, kv, dim, q_off
        first = shared // PAGE
        own = [-(-m // PAGE) if m > 0 else 0 for _, m in lens]
        pages = first + sum(own) + spare
        self.width = max(first + max(own) + table_spare, 1)
        order = torch.randperm(pages, generator=g)
        self.table = torch.randint(-5, 10 ** 6, (len(lens), self.width), generator=g).to(torch.int32)     # (what lies behind a sequence is anything)
        k = torch.full((pages, kv, PAGE, dim), float("nan"))
        v = torch.full((pages, kv, dim, PAGE), float("nan"))
        at = first
        k[order[:first]] = torch.randn(first, kv, PAGE, dim, generator=g) * spread
        v[order[:first]] = torch.randn(first, kv, dim, PAGE, generator=g)
        for b, n in enumerate(own):
            self.table[b, :first] = order[:first]
            self.table[b, first:first + n] = order[at:at + n]
            for i in range(n):
                held = min(PAGE, lens[b][1] - i * PAGE)
                k[order[at + i], :, :held] = torch.randn(kv, held, dim, generator=g) * spread
                v[order[at + i], :, :, :held] = torch.randn(kv, dim, held, generator=g)
            at += n
        self.k, self.v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        self.counts = [n for n, _ in lens]
        self.tokens = sum(self.counts) + pad_rows
        self.qkv = torch.randn(self.tokens, q_off + (heads + 2 * kv) * dim, generator=g).to(torch.bfloat16)
        self.pos = [shared + m - n + i for n, m in lens for i in range(n)] + [7] * pad_rows
        self.max_len, self.max_new = max(1, shared + max(m for _, m in lens)), max(self.counts)
        self.scale = dim ** -0.5

    def run(self, ops, **change):
        a = dict(k=guarded(self.k), v=guarded(self.v), qkv=guarded(self.qkv), shared=self.shared, max_len=self.max_len)
        a.update(change)
        return ops.attention_shared_bf16(a["qkv"], a["k"], a["v"], i32(starts(self.counts)), i32(self.pos), guarded(self.table), len(self.lens),
                                         self.max_new, a["shared"], a["max_len"], self.heads, self.kv, self.dim, self.scale, self.q_off)

    def plain(self):
        """(result, sum of weights times |v|) in 64 bits."""
        heads, kv, dim, per = self.heads, self.kv, self.dim, self.heads // self.kv
        out, size, at = np.zeros((self.tokens, heads, dim)), np.zeros((self.tokens, heads, dim)), 0
        q = self.qkv[:, self.q_off:self.q_off + heads * dim].double().view(self.tokens, heads, dim).numpy()
        for b, (new, _) in enumerate(self.lens):
            pages = self.table[b, :-(-(max(self.pos[at:at + new], default=-1) + 1) // PAGE)].long()
            for h in range(kv if new else 0):
                keys = self.k[pages, h].reshape(-1, dim).double().numpy()
                values = self.v[pages, h].transpose(1, 2).reshape(-1, dim).double().numpy()
                for i in range(at, at + new):
                    length, own = self.pos[i] + 1, slice(h * per, h * per + per)
                    s = q[i, own] @ keys[:length].T * self.scale
                    w = np.exp(s - s.max(1, keepdims=True))
                    w /= w.sum(1, keepdims=True)
                    out[i, own], size[i, own] = w @ values[:length], w @ np.abs(values[:length])
            at += new
        return out.reshape(self.tokens, -1), size.reshape(self.tokens, -1)

    def check(self, got):
        """A weight is rounded to bfloat16 once (half a step of itself), so the sum of weighted values is off by that share of the
        sum of weights times |v| at most; the result is rounded once; float32 scores of |s| < 2^6 are off by 2^-16 at most with the
        128 additions of a dot product and the exponential's own, which a weight is off by relative to itself."""
        want, size = self.plain()
        bound = BF16_STEP * np.abs(want) + (BF16_STEP + 2.0 ** -14) * size + 1e-30
        got = f64(got)
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


SHARED = [  # lens, shared, heads, kv, dim
    ([(1, 1)], 32, 2, 1, 32), ([(1, 33), (1, 5)], 64, 4, 2, 64), ([(1, 31), (1, 32), (1, 64)], 96, 8, 2, 128),
    ([(1, 40)] * 5, 0, 4, 4, 64), ([(3, 3), (1, 70), (5, 20), (2, 2)], 160, 6, 2, 64), ([(7, 30), (7, 7)], 32, 5, 1, 128),
    ([(1, 600), (1, 512), (1, 513), (2, 1025)], 32, 2, 2, 32), ([(4, 9)], 640, 3, 3, 128), ([(1, 3)] * 20, 288, 4, 1, 64),
    # (from 33 columns of a key head on the pages go through LDS, tiles of 64 and, from 65 on, 128; an odd last page, one pair, one page)
    ([(1, 2)] * 5, 288, 8, 1, 128), ([(2, 3)] * 5, 96, 8, 1, 128), ([(1, 1)] * 6, 32, 6, 1, 64), ([(3, 5)] * 15, 608, 3, 1, 32),
    ([(1, 4)] * 17, 544, 16, 2, 64), ([(2, 500), (0, 33), (1, 1)], 512, 8, 1, 128), ([(1, 2)] * 70, 64, 1, 1, 32), ([(40, 40), (9, 100)], 64, 4, 2, 64),
    # no sequence, one without a new token, first and last
    ([(0, 0), (2, 40), (0, 70)], 64, 4, 2, 64), ([(0, 5), (0, 0), (1, 3), (0, 0)], 224, 40, 1, 32),
]
if not EMULATED:                          # runs of more than sixteen pages: from 129 columns on by eight wavefronts
    SHARED += [([(3, 3)] * 6, 20480, 64, 8, 64), ([(2, 40), (1, 1)] * 6, 9600, 128, 8, 128), ([(20, 22)] * 7, 17472, 8, 8, 32),
               ([(1, 50)] * 3, 33056, 16, 8, 128)]


@pytest.mark.parametrize("lens, shared, heads, kv, dim", SHARED)
def test_attention_over_shared_pages(ops, lens, shared, heads, kv, dim):
    c = SharedCase(lens, shared, heads, kv, dim)
    c.check(c.run(ops))


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attention_over_shared_pages_reads_its_columns_and_leaves_rows_behind_the_sequences_at_zero(ops, dim):
    c = SharedCase([(2, 10), (1, 35)], 64, 4, 2, dim, q_off=2 * dim, pad_rows=3, seed=3)
    got = c.run(ops)
    assert (f64(got)[3:] == 0).all()
    c.check(got)


@pytest.mark.parametrize("heads", [4, 40])
def test_attention_over_shared_pages_keeps_what_pads_a_batch_to_itself(ops, heads):
    """Rows that are no sequence's hold NaN at positions that are none; the others are what they are without them."""
    c = SharedCase([(2, 10), (1, 35)], 96, heads, 2, 64, pad_rows=3, seed=8)
    c.qkv[3:] = float("nan")
    c.pos[3:] = [-1, -7, 10 ** 9]
    got = f64(c.run(ops))
    assert (got[3:] == 0).all()
    c.check(torch.tensor(got))


@pytest.mark.parametrize("rows, n", [(3, 40), (20, 40), (16, 9000)])
def test_products_in_4_bits_keep_an_infinity_to_its_row(ops, rows, n):
    if EMULATED:
        n = 40
    x, code, packed, scales, zero = int4_inputs(rows, n, 512, 64, True, torch.bfloat16, False, 4)
    args = guarded(packed), guarded(scales), 64, guarded(zero), torch.float32
    want = f64(ops.gemm_int4_bf16(guarded(x), *args))
    x[1, 70], x[2, 9] = float("inf"), float("nan")
    got = f64(ops.gemm_int4_bf16(guarded(x), *args))
    others = np.arange(rows) > 2
    others[0] = True
    assert np.array_equal(got[others], want[others]) and not np.isfinite(got[1:3]).any()


def test_attention_over_shared_pages_of_tokens_within_them(ops):
    """A token whose position lies among the shared tokens sees the keys up to its own."""
    c = SharedCase([(1, 5), (2, 40)], 96, 4, 2, 64, seed=4)
    c.pos = [50, 95, 96 + 39]
    c.check(c.run(ops))
    for heads in (12, 24):                                    # columns of a key head: 36 and 72
        c = SharedCase([(1, 5), (2, 40)], 224, heads, 1, 32, seed=4)
        c.pos = [70, 191, 224 + 39]
        c.check(c.run(ops))


def test_attention_over_shared_pages_finds_one_far_key(ops):
    """All queries look along one direction and one key, the first or the last of a page, lies far along it."""
    c = SharedCase([(1, 70), (1, 1)], 320, 2, 1, 64, seed=5)
    for at in (0, 31, 32, 288, 319):
        k = c.k.clone()
        page, row = int(c.table[0, at // PAGE]), at % PAGE
        q = c.qkv[:, :128].float().view(2, 2, 64)
        k[page, 0, row] = (q[0, 1] * 4).to(torch.bfloat16)
        kept, c.k = c.k, k
        c.check(c.run(ops))
        c.k = kept


def test_attention_over_shared_pages_does_not_depend_on_the_bound(ops):
    """A larger max_len makes a larger grid, the same sums in the same order."""
    c = SharedCase([(1, 40), (3, 600)], 64, 4, 2, 64, seed=6, table_spare=60)
    assert torch.equal(c.run(ops), c.run(ops, max_len=c.max_len + 1500))


def test_attention_over_shared_pages_refuses_what_it_does_not_take(ops):
    from rust_inference_amd.errors import InferenceError
    c = SharedCase([(1, 5), (1, 9)], 64, 4, 2, 64)
    for change in (dict(shared=33), dict(shared=-32), dict(shared=64 + 32 * c.width), dict(max_len=32 * c.width + 1), dict(max_len=0),
                   dict(qkv=guarded(c.qkv.float())), dict(k=guarded(c.k[:, :1])), dict(qkv=guarded(c.qkv[:, :200]))):
        with pytest.raises(InferenceError):
            c.run(ops, **change)
    for name, value in (("dim", 48), ("heads", 5), ("q_off", 4), ("scale", 0.0), ("scale", float("inf")), ("max_new", 0)):
        kept = getattr(c, name)
        setattr(c, name, value)
        with pytest.raises(InferenceError):
            c.run(ops)
        setattr(c, name, kept)


@pytest.mark.skipif(EMULATED, reason="nine gigabytes of pages")
def test_attention_over_shared_pages_whose_offsets_pass_32_bits(ops):
    pages, kv, dim = 70000, 8, 128
    k = torch.empty((pages, kv, PAGE, dim), dtype=torch.bfloat16, device=DEV)
    v = torch.empty((pages, kv, dim, PAGE), dtype=torch.bfloat16, device=DEV)
    c = SharedCase([(1, 5), (2, 40)], 96, 16, kv, dim, seed=7)
    used = c.k.shape[0]
    k[pages - used:], v[pages - used:] = c.k.to(DEV), c.v.to(DEV)
    small = c.run(ops)
    c.table = torch.where((c.table >= 0) & (c.table < used), c.table + (pages - used), c.table)
    got = c.run(ops, k=k, v=v)
    assert torch.equal(got, small)


# ---------------------------------------------------------------- drafted tokens
def softmax(x, temperature):
    x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), np.finfo(np.float32).max))
    if not np.isfinite(x).any():
        return np.zeros_like(x)
    w = np.exp((x - x.max()) / temperature)
    return w / w.sum()


def plain_verify(logits, draft, tokens, counts, u, temperature, margin=1e-10):
    """(accepted, out) sequence by sequence in 64 bits; asserts that no number lies within ``margin`` of a border, where the kernel
    (exponentials to 3e-13, sums of up to 2^18 of them to 2^-35 at worst, 3e-11) could rightly decide otherwise."""
    cu = starts(counts)
    accepted, out = [], np.full(len(tokens), -1)
    vocab = logits.shape[1]
    for r0, r1 in zip(cu[:-1], cu[1:]):
        if r0 == r1:
            accepted.append(0)
            continue
        stop = r1 - 1
        weights = None
        for r in range(r0, r1 - 1):
            d = int(tokens[r + 1])
            if temperature <= 0:
                row = np.where(np.isnan(logits[r]), -np.inf, logits[r])
                if int(row.argmax()) != d:
                    stop = r
                    break
                continue
            p = softmax(logits[r], temperature)
            q = softmax(draft[r + 1], temperature) if draft is not None else None
            known = 0 <= d < vocab
            qd, pd = (q[d] if known else 0.0) if q is not None else 1.0, p[d] if known else 0.0
            side = float(u[r]) * qd - pd
            assert abs(side) > margin * max(pd, 1e-300) or (qd == 0 and pd == 0) or u[r] == 0
            if not side < 0:
                stop = r
                if q is not None:
                    weights = np.maximum(p - q, 0.0)
                else:
                    weights = p.copy()
                    if known:
                        weights[d] = 0.0
                if not weights.sum() > 0:
                    weights = p
                break
        accepted.append(stop - r0)
        out[r0:stop] = tokens[r0 + 1:stop + 1]
        if temperature <= 0:
            out[stop] = int(np.where(np.isnan(logits[stop]), -np.inf, logits[stop]).argmax())
            continue
        if weights is None:
            weights = softmax(logits[stop], temperature)
        upto = np.cumsum(weights)
        target = float(u[r1 - 1]) * upto[-1]
        assert np.abs(upto[:-1][weights[:-1] > 0] - target).min(initial=1.0) > margin * max(upto[-1], 1e-300) or target == 0
        past = np.nonzero(upto > target)[0]
        some = np.nonzero(weights > 0)[0]
        out[stop] = past[0] if len(past) else some[-1] if len(some) else 0
    return np.array(accepted), out


def drafted(counts, vocab, temperature, with_draft, seed=0, noise=0.7):
    rng = np.random.default_rng(seed)
    rows = int(sum(counts))
    logits = (2.0 * rng.standard_normal((rows, vocab))).astype(np.float32)
    draft = np.roll(logits, 1, 0) + noise * rng.standard_normal((rows, vocab)).astype(np.float32)
    t = temperature if temperature > 0 else 0.05
    tokens = np.array([rng.choice(vocab, p=softmax(row, t)) for row in draft])
    return logits, (draft.astype(np.float32) if with_draft else None), tokens, rng.random(rows).astype(np.float32)


def verify(ops, logits, draft, tokens, counts, u, temperature):
    t = lambda a: None if a is None else guarded(torch.tensor(np.ascontiguousarray(a), dtype=torch.float32))  # noqa: E731
    accepted, out = ops.verify_drafts(t(logits), i32(tokens), i32(starts(counts)), t(u), temperature, t(draft))
    return accepted.cpu().numpy(), out.cpu().numpy()


def same(got, want):
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (got, want)


VERIFY = [([1], 7), ([3, 1, 2], 411), ([5] * 6, 1000), ([0, 4, 0, 0, 9, 1, 0], 64), ([2, 6], 4096), ([6, 2], 4097), ([3, 3], 9002), ([70, 2], 33),
          ([1, 1], 1), ([4, 2], 3)]


@pytest.mark.parametrize("counts, vocab", VERIFY)
@pytest.mark.parametrize("temperature, with_draft", [(1.0, True), (0.6, True), (1.3, False), (0.0, False), (-1.0, True)])
def test_drafts_are_verified(ops, counts, vocab, temperature, with_draft):
    for seed in range(2):
        logits, draft, tokens, u = drafted(counts, vocab, temperature, with_draft, seed)
        same(verify(ops, logits, draft, tokens, counts, u if temperature > 0 else None, temperature),
             plain_verify(logits, draft, tokens, counts, u, temperature))


@pytest.mark.parametrize("temperature", [1e-30, 1e-12, 1e-8, 1e-6, 1e-3, 50.0, 1e6, 1e30])
@pytest.mark.parametrize("with_draft", [True, False])
def test_temperatures_at_the_ends_of_their_range(ops, temperature, with_draft):
    """Cold: everything falls to the largest logit; hot: all entries weigh alike."""
    counts, vocab = [3, 2, 5], 4500
    logits, draft, tokens, u = drafted(counts, vocab, 1.0, with_draft, 12)
    best = logits.argmax(1)
    tokens[1], tokens[6], tokens[7] = best[0], best[5], best[6]
    if with_draft:
        draft[[1, 6, 7], tokens[[1, 6, 7]]] = 9.0
    with np.errstate(over="ignore"):
        want = plain_verify(logits, draft, tokens, counts, u, temperature, margin=1e-9)
    same(verify(ops, logits, draft, tokens, counts, u, temperature), want)


@pytest.mark.parametrize("temperature", [1e33, 1e35, 3e36, 1e38, 1e300])
@pytest.mark.parametrize("large", [False, True])
def test_very_high_temperatures_with_masked_entries(ops, temperature, large):
    """Logits as large as the temperature, up to float32's ends, or ordinary ones beside it; what is masked weighs nothing still."""
    counts, vocab = [3, 2, 5], 4500
    rng = np.random.default_rng(13)
    logits, draft, tokens, u = drafted(counts, vocab, 1.0, True, 13)
    if large:
        logits, draft = (np.clip(0.5 * a.astype(np.float64) * min(temperature, 1e38), -3.4e38, 3.4e38).astype(np.float32) for a in (logits, draft))
    for a in (logits, draft):
        a[rng.random(a.shape) < 0.4] = -np.inf
        a[rng.random(a.shape) < 0.1] = np.nan
    for d in (draft, None):
        same(verify(ops, logits, d, tokens, counts, u, temperature), plain_verify(logits, d, tokens, counts, u, temperature, margin=1e-9))


@pytest.mark.parametrize("vocab", [411, 5000])
def test_drafts_of_the_target_itself_all_stand(ops, vocab):
    counts = [6, 1, 9]
    logits, _, tokens, u = drafted(counts, vocab, 1.0, True, 3)
    draft = np.roll(logits, 1, 0)
    accepted, out = verify(ops, logits, draft, tokens, counts, u, 1.0)
    assert accepted.tolist() == [5, 0, 8]
    same((accepted, out), plain_verify(logits, draft, tokens, counts, u, 1.0, margin=0.0))


def test_masked_entries_rows_and_drafts_outside_the_vocabulary(ops):
    counts, vocab = [4, 3, 3, 2, 2], 500
    logits, draft, tokens, u = drafted(counts, vocab, 0.9, True, 5)
    rng = np.random.default_rng(6)
    cut = rng.random(logits.shape) < 0.9
    logits[cut] = -np.inf
    draft[rng.random(draft.shape) < 0.5] = -np.inf
    logits[:, ::17] = np.nan
    draft[starts(counts)[:-1]] = np.nan                      # rows of tokens that are no drafts: not read
    logits[5] = -np.inf                                      # a row that masks everything
    logits[7, 100] = np.inf
    tokens[8], tokens[11] = -3, vocab
    want = plain_verify(logits, draft, tokens, counts, u, 0.9)
    same(verify(ops, logits, draft, tokens, counts, u, 0.9), want)
    same(verify(ops, logits, None, tokens, counts, u, 0.9), plain_verify(logits, None, tokens, counts, u, 0.9))
    same(verify(ops, logits, None, tokens, counts, None, 0.0), plain_verify(logits, None, tokens, counts, u, 0.0))
    masked = np.full((2, 4500), -np.inf, dtype=np.float32)
    for t in (0.0, 1.0):
        accepted, out = verify(ops, masked, None, np.array([3, 4]), [2], np.array([0.5, 0.5]), t)
        assert accepted.tolist() == [0] and out.tolist() == [0, -1]


def test_numbers_at_the_ends_of_their_range(ops):
    """0 lets every draft of the target's stand and draws the first token that weighs anything; a number that is not below 1 draws
    the last such token."""
    counts, vocab = [3, 2, 1], 4200
    logits, draft, tokens, u = drafted(counts, vocab, 1.0, True, 8)
    logits[:, 0], logits[:, -1], logits[:, 4097:] = -np.inf, -np.inf, -np.inf
    tokens = np.minimum(tokens, 4000) + 1
    accepted, out = verify(ops, logits, draft, tokens, counts, 0 * u, 1.0)
    assert accepted.tolist() == [2, 1, 0] and out[[2, 4, 5]].tolist() == [1, 1, 1]
    accepted, out = verify(ops, logits, None, tokens, counts, 0 * u + 1.0, 1.0)
    assert accepted.tolist() == [0, 0, 0] and out.tolist() == [4096, -1, -1, 4096, -1, 4096]


def test_greedy_takes_the_first_of_equal_ones(ops):
    logits = np.zeros((4, 9000), dtype=np.float32)
    logits[0, [5, 8000]], logits[1, [4096, 4095]], logits[2, 8999] = 3.0, 2.0, 1.0
    logits[3, 1:] = -1.0
    accepted, out = verify(ops, logits, None, np.array([0, 5, 4095, 8998]), [4], None, 0.0)
    assert accepted.tolist() == [2] and out.tolist() == [5, 4095, 8999, -1]


def test_rows_behind_the_sequences_and_sequences_behind_the_rows(ops):
    logits, draft, tokens, u = drafted([3, 2, 4], 300, 1.0, True, 9)
    t = lambda a: guarded(torch.tensor(np.ascontiguousarray(a), dtype=torch.float32))  # noqa: E731
    for temperature in (1.0, 0.0):
        want = plain_verify(logits[:5], draft[:5], tokens[:5], [3, 2], u[:5], temperature)
        accepted, out = ops.verify_drafts(t(logits), i32(tokens), i32([0, 3, 5]), t(u), temperature, t(draft))
        assert np.array_equal(accepted.cpu().numpy(), want[0])
        assert out.cpu().numpy().tolist() == want[1].tolist() + [-1] * 4
        accepted, out = ops.verify_drafts(t(logits), i32(tokens), i32([-4, 3, 50, 60]), t(u), temperature, t(draft))      # held to the rows
        want = plain_verify(logits, draft, tokens, [3, 6], u, temperature)
        assert np.array_equal(accepted.cpu().numpy(), want[0].tolist() + [0]) and np.array_equal(out.cpu().numpy(), want[1])


def test_what_is_put_out_is_distributed_as_the_target(ops):
    """Every pair of numbers of a grid and every draft, weighed by the draft's distribution: the first token put out has the target's
    probabilities, up to the grid: each of the two draws is off by at most one of its cells per border, vocab borders in all."""
    vocab, grid = 5, 6 if EMULATED else 64
    rng = np.random.default_rng(10)
    p_row, q_row = rng.standard_normal((2, vocab)).astype(np.float32)
    cells = [(d, a, b) for d in range(vocab) for a in range(grid) for b in range(grid)]
    rows = 2 * len(cells)
    logits = np.tile(p_row, (rows, 1))
    draft = np.tile(q_row, (rows, 1))
    tokens = np.array([[0, d] for d, _, _ in cells]).reshape(-1)
    u = np.array([[(a + 0.5) / grid, (b + 0.5) / grid] for _, a, b in cells]).reshape(-1)
    _, out = verify(ops, logits, draft, tokens, [2] * len(cells), u, 1.0)
    weight = np.repeat(softmax(q_row, 1.0), grid * grid) / grid ** 2
    found = np.bincount(out[::2], weights=weight, minlength=vocab)
    assert np.abs(found - softmax(p_row, 1.0)).max() <= 2.0 / grid


def test_drafts_are_refused_where_an_operand_does_not_fit(ops):
    from rust_inference_amd.errors import InferenceError
    logits, draft, tokens, u = drafted([3, 2], 40, 1.0, True)
    t = lambda a: guarded(torch.tensor(np.ascontiguousarray(a), dtype=torch.float32))  # noqa: E731
    good = dict(logits=t(logits), tokens=i32(tokens), cu=i32([0, 3, 5]), u=t(u), temperature=1.0, draft=t(draft))
    for change in (dict(u=None), dict(u=t(u[:4])), dict(tokens=i32(tokens[:4])), dict(tokens=guarded(torch.tensor(tokens))), dict(draft=t(draft[:4])),
                   dict(draft=t(draft[:, :39])), dict(logits=t(logits).double()), dict(logits=t(logits)[0]), dict(cu=i32([0])),
                   dict(logits=t(logits)[:0]), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(logits=t(np.concatenate([logits, logits], 1))[:, :40])):
        a = dict(good, **change)
        with pytest.raises(InferenceError):
            ops.verify_drafts(a["logits"], a["tokens"], a["cu"], a["u"], a["temperature"], a["draft"])


# ---------------------------------------------------------------- devices, streams, graphs, together
@pytest.mark.skipif(EMULATED, reason="two devices")
def test_operands_on_two_devices_are_refused(ops):
    from rust_inference_amd.errors import InferenceError
    x, _, packed, scales, zero = int4_inputs(2, 16, 128, 32, True, torch.bfloat16, False)
    c = SharedCase([(1, 5)], 64, 4, 2, 64)
    logits, draft, tokens, u = drafted([3], 40, 1.0, True)
    t = lambda a: torch.tensor(a, dtype=torch.float32)  # noqa: E731
    for call in (lambda: ops.gemm_int4_bf16(x, packed, scales, 32, zero), lambda: ops.gemm_int4_bf16(x.to(DEV), packed.to(DEV), scales, 32),
                 lambda: ops.gemm_int4_bf16(x.to(DEV), packed.to(DEV), scales.to(DEV), 32, zero), lambda: c.run(ops, k=c.k),
                 lambda: c.run(ops, qkv=c.qkv), lambda: ops.verify_drafts(t(logits), i32(tokens), i32([0, 3]), t(u).to(DEV), 1.0),
                 lambda: ops.verify_drafts(t(logits).to(DEV), i32(tokens), i32([0, 3]), t(u), 1.0),
                 lambda: ops.verify_drafts(t(logits).to(DEV), i32(tokens), i32([0, 3]), t(u).to(DEV), 1.0, t(draft))):
        with pytest.raises(InferenceError):
            call()


@pytest.mark.skipif(EMULATED, reason="streams and graphs")
def test_on_another_stream_and_in_two_graphs_that_are_replayed_in_turn(ops):
    """Each operator on a stream of its own, and two captured graphs of all three whose inputs change between the replays: every
    replay gives the eager bits."""
    def inputs(seed):
        c = SharedCase([(2, 40), (1, 600), (3, 3)], 128, 8, 2, 64, seed=seed)
        x, _, packed, scales, zero = int4_inputs(6, 40, 512, 64, True, torch.bfloat16, False, seed)
        logits, draft, tokens, u = drafted([2, 1, 3], 5000, 1.0, True, seed)
        f = lambda a: torch.tensor(a, dtype=torch.float32, device=DEV)  # noqa: E731
        return c, [a.to(DEV) for a in (c.qkv, c.k, c.v, x, packed, scales, zero)] + [f(logits), f(draft), f(u), i32(tokens)]

    def call(c, a, table, pos, cu):
        return [ops.attention_shared_bf16(a[0], a[1], a[2], cu, pos, table, 3, 3, 128, 728, 8, 2, 64, 0.125),
                ops.gemm_int4_bf16(a[3], a[4], a[5], 64, a[6]), ops.gemm_int4_bf16(a[3], a[4], a[5], 64, None, torch.float32),
                *ops.verify_drafts(a[7], a[10], cu, a[9], 0.8, a[8]), *ops.verify_drafts(a[7], a[10], cu, None, 0.0)]

    cases = [inputs(seed) for seed in (21, 22, 23)]
    eager = []
    for c, a in cases:
        table, pos, cu = c.table.to(DEV), i32(c.pos), i32(starts(c.counts))
        eager.append([t.clone() for t in call(c, a, table, pos, cu)])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for (c, a), want in zip(cases, eager):
            side.wait_stream(torch.cuda.default_stream())
            got = call(c, a, c.table.to(DEV), i32(c.pos), i32(starts(c.counts)))
            side.synchronize()
            assert all(torch.equal(g, w) for g, w in zip(got, want))
    graphs = []
    for _ in range(2):
        c, a = cases[0]
        held = [t.clone() for t in a]
        table, pos, cu = c.table.to(DEV), i32(c.pos), i32(starts(c.counts))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(c, held, table, pos, cu)
        graphs.append((graph, held, table, out, pos, cu))      # (what a graph reads lives as long as it)
    for turn in range(6):
        for i, (graph, held, table, out, *_) in enumerate(graphs):
            which = (turn + i) % 3
            for h, t in zip(held, cases[which][1]):
                h.copy_(t)
            table.copy_(cases[which][0].table.to(DEV))
            graph.replay()
        torch.ones(1000, device=DEV).sum()
        torch.cuda.synchronize()
        for i, (graph, held, table, out, *_) in enumerate(graphs):
            assert all(torch.equal(g, w) for g, w in zip(out, eager[(turn + i) % 3])), (turn, i)


def test_a_drafted_step_from_weights_to_tokens(ops):
    """The three as they follow one another: attention of a drafted step over a shared prompt, the target's logits from it through a
    matrix in 4 bits, the draft's logits through another, the draft's tokens sampled from them, the verification; each against the
    plain operator on what it was given."""
    counts, shared, vocab = [3, 1, 4], 96, 300
    c = SharedCase([(n, n + 20 + 9 * i) for i, n in enumerate(counts)], shared, 4, 2, 64, seed=31)
    attended = c.run(ops)
    c.check(attended)
    _, code, packed, scales, zero = int4_inputs(1, vocab, 256, 64, True, torch.float32, False, 32)
    scales = scales * 30
    logits = ops.gemm_int4_bf16(attended, guarded(packed), guarded(scales), 64, guarded(zero), torch.float32)
    xd, w, s, z = plain_int4(attended.cpu(), code, scales, zero, 64)
    assert (np.abs(f64(logits) - xd @ w.T) <= F32_STEP * 200 * (np.abs(xd) @ (s * (32.0 + code.numpy() + z)).T)).all()
    x = guarded(torch.randn(8, 256, generator=torch.Generator().manual_seed(33)).to(torch.bfloat16))
    draft = ops.gemm_int4_bf16(x, guarded(packed), guarded(scales * 0.1), 64, None, torch.float32)
    u = np.random.default_rng(34).random((2, 8)).astype(np.float32)
    tokens = ops.sample(draft, guarded(torch.tensor(u[0])), 0.9)
    accepted, out = ops.verify_drafts(logits, tokens, i32(starts(counts)), guarded(torch.tensor(u[1])), 0.9, draft)
    want = plain_verify(f64(logits).astype(np.float32), f64(draft).astype(np.float32), tokens.cpu().numpy(), counts, u[1], 0.9)
    same((accepted.cpu().numpy(), out.cpu().numpy()), want)
