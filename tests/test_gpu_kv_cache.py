"""The paged key/value cache on the GPU against 64-bit sums (tests/kv_ref.py): append, read, attention."""
import dataclasses
import math

import numpy as np
import pytest

import kv_ref as ref
from litenn_b200 import capi

pytestmark = pytest.mark.gpu

FMTS = [ref.Q4_0, ref.Q8_0, ref.F16]


@pytest.fixture(scope="module", autouse=True)
def device(qmm_lib):
    import torch
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    capi.kernel_status(0)


def torch_of(x, bf16=False):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t.bfloat16() if bf16 else t


def np_of(t):
    return t.float().cpu().numpy()


@dataclasses.dataclass
class Paged:
    """A pool with shuffled pages and sequences of given lengths; every byte that no append has written is 0xFF."""
    fmt: int
    kv_heads: int
    hd: int
    page: int
    lens: list
    spare: int = 2
    seed: int = 0

    def __post_init__(self):
        import torch
        rng = np.random.default_rng(self.seed)
        self.width = max(1, max(-(-n // self.page) for n in self.lens))
        used = sum(-(-n // self.page) for n in self.lens)
        self.n_pages = used + self.spare
        order = rng.permutation(self.n_pages)[:used].tolist()
        table = np.full((len(self.lens), self.width), 2 ** 30, dtype=np.int32)  # what lies past a length is not read
        for s, n in enumerate(self.lens):
            for i in range(-(-n // self.page)):
                table[s, i] = order.pop()
        self.table = table
        nbytes = capi.kv_pool_bytes(self.fmt, self.kv_heads, self.hd, self.page, self.n_pages)
        self.pool = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
        self.cache = capi.KVCache(self.fmt, self.kv_heads, self.hd, self.page, self.n_pages, self.pool.data_ptr())
        self.table_dev = torch_of(table)
        self.workspace = torch.zeros(capi.KV_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
        self.hold = []

    def batch(self, rows, lens, total=None, single=False):
        begin = torch_of(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
        length = torch_of(np.asarray(lens, dtype=np.int32))
        self.hold += [begin, length]
        return capi.KVBatch(len(lens), self.width, self.table_dev.data_ptr(), length.data_ptr(),
                            0 if single else begin.data_ptr(), sum(rows) if total is None else total)

    def fill(self, rng, k_scale=1.0):
        """Appends random keys and values up to the lengths, without rotation; the values that the cache holds."""
        rows = list(self.lens)
        k = (rng.standard_normal((sum(rows), self.kv_heads, self.hd)) * k_scale).astype(np.float32)
        v = rng.standard_normal((sum(rows), self.kv_heads, self.hd)).astype(np.float32)
        kd, vd, w = torch_of(k), torch_of(v), self.kv_heads * self.hd
        self.cache.append(self.batch(rows, rows), None, 0, 0, 0, 0, kd.data_ptr(), w, vd.data_ptr(), w, 0, 0, 0)
        assert capi.kernel_status(0) == 0
        cut = np.cumsum(rows)[:-1]
        return np.split(ref.stored(k, self.fmt), cut), np.split(ref.stored(v, self.fmt), cut)

    def attend(self, q, rows, lens, heads, bf16=False, out_bf16=False, window=0, single=False, scale=None, total=None,
               prompt=False):
        import torch
        asked = len(q)
        if prompt:  # rows behind the last sequence, so that the call is one of many
            total = max(len(q), -(-4096 // heads))
            q = np.concatenate([q, np.ones((total - len(q), *q.shape[1:]), q.dtype)])
        qd = torch_of(q.reshape(len(q), -1), bf16)
        out = torch.full((len(q), heads * self.hd), 7.0, device="cuda", dtype=torch.bfloat16 if out_bf16 else torch.float32)
        self.cache.attend(self.batch(rows, lens, total, single), heads, qd.data_ptr(), int(bf16), heads * self.hd,
                          out.data_ptr(), int(out_bf16), heads * self.hd, self.hd ** -0.5 if scale is None else scale, window,
                          self.workspace.data_ptr())
        assert capi.kernel_status(0) == 0
        assert (out[asked:] == 7.0).all()
        return np_of(out)[:asked].reshape(asked, heads, self.hd).astype(np.float64)


def check_attention(p, rows, lens, heads, rng, bf16=False, out_bf16=False, window=0, single=False, q_scale=2.0, half=False):
    ks, vs = p.fill(rng)
    q = (rng.standard_normal((sum(rows), heads, p.hd)) * q_scale).astype(np.float32)
    if bf16:
        q = ref.bf16_round(q)
    got = p.attend(q, rows, lens, heads, bf16, out_bf16, window, single)
    at = 0
    for s, (n, r) in enumerate(zip(lens, rows)):
        if r == 0:
            continue
        want = ref.attention(q[at:at + r], ks[s], vs[s], n, p.hd ** -0.5, window)
        bound = ref.attention_bound(q[at:at + r], ks[s], vs[s], p.hd ** -0.5, out_bf16, half)
        err = np.abs(got[at:at + r] - want).max()
        assert err <= bound, (s, n, r, err, bound)
        at += r


# ---- append and read ----------------------------------------------------------------------------------------------------

def check_append(fmt, hd, heads, kv_heads, page, rope_dim, halves, bf16, rows, lens):
    import torch
    rng = np.random.default_rng(hd + page)
    p = Paged(fmt, kv_heads, hd, page, lens)
    before = p.pool.clone()
    width = heads + 2 * kv_heads
    qkv = rng.standard_normal((sum(rows) + 3, width, hd)).astype(np.float32) * 3  # three rows behind the last sequence
    qkv[0, heads] = 0.0                       # a block of zeros
    qkv[1, heads + kv_heads, :32] = np.where(np.arange(32) % 5, 1.0, -2.5)  # equals of both signs
    if bf16:
        qkv = ref.bf16_round(qkv)
    x = torch_of(qkv.reshape(len(qkv), -1), bf16)
    freq, gain = capi.rope_frequencies(rope_dim or 2, 10000.0)
    freq_dev = torch_of(freq)
    rope = capi.Rope(rope_dim, int(halves), freq_dev.data_ptr(), 1.25) if rope_dim else None
    q_out = torch.full((len(qkv), heads * hd), 9.0, device="cuda", dtype=x.dtype)
    at, item, stride = x.data_ptr(), x.element_size(), width * hd
    b = p.batch(rows, lens, total=len(qkv))
    p.cache.append(b, rope, heads, int(bf16), at, stride, at + heads * hd * item, stride, at + (heads + kv_heads) * hd * item,
                   stride, q_out.data_ptr(), int(bf16), heads * hd)
    k_out = torch.full((len(qkv), kv_heads * hd), 9.0, device="cuda")
    v_out = k_out.clone()
    p.cache.read(b, k_out.data_ptr(), kv_heads * hd, v_out.data_ptr(), kv_heads * hd, 0)
    assert capi.kernel_status(0) == 0
    pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)])
    n = len(pos)
    want_q = ref.rotate(qkv[:n, :heads], pos, freq, 1.25, rope_dim, halves)
    want_k = ref.stored(ref.rotate(qkv[:n, heads:heads + kv_heads], pos, freq, 1.25, rope_dim, halves), fmt)
    want_v = ref.stored(qkv[:n, heads + kv_heads:], fmt)
    np.testing.assert_array_equal(np_of(q_out)[:n].reshape(want_q.shape), ref.bf16_round(want_q) if bf16 else want_q)
    np.testing.assert_array_equal(np_of(k_out)[:n].reshape(want_k.shape), want_k.astype(np.float32))
    np.testing.assert_array_equal(np_of(v_out)[:n].reshape(want_v.shape), want_v.astype(np.float32))
    for t in (q_out, k_out, v_out):
        assert (t[n:] == 9.0).all()           # rows behind the last sequence
    # the bytes lie where the header says, and nothing else was written
    tb = ref.tile_bytes(fmt, hd)
    pool = p.pool.cpu().numpy().reshape(p.n_pages, kv_heads, page // 16, tb)
    seq = np.repeat(np.arange(len(rows)), rows)
    for i in rng.choice(n, 6, replace=False):
        for h in range(kv_heads):
            tile = pool[p.table[seq[i], pos[i] // page], h, pos[i] % page // 16]
            for d in rng.choice(hd, 8, replace=False):
                assert np.float32(ref.tile_value(tile, fmt, hd, True, pos[i] % 16, d)) == np.float32(want_k[i, h, d])
                assert np.float32(ref.tile_value(tile, fmt, hd, False, pos[i] % 16, d)) == np.float32(want_v[i, h, d])
    written = n * kv_heads * tb // 16
    changed = int((p.pool != before).sum())
    assert changed <= written and changed > written // 2


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,heads,kv_heads,page,rope_dim,halves,bf16", [
    (128, 8, 2, 16, 128, False, False), (128, 4, 4, 64, 64, True, True), (64, 3, 1, 32, 64, True, False),
    (96, 6, 3, 48, 96, True, False), (96, 2, 1, 16, 34, False, True), (256, 2, 2, 128, 256, True, False),
    (256, 4, 1, 16, 0, False, False), (64, 2, 2, 16, 8, True, True)])
def test_append_stores_what_the_rules_say(fmt, hd, heads, kv_heads, page, rope_dim, halves, bf16):
    check_append(fmt, hd, heads, kv_heads, page, rope_dim, halves, bf16, [5, 0, 1, 40], [21, 7, 1, 140])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,heads,kv_heads,page,rope_dim,halves,bf16", [
    (128, 17, 9, 32, 128, False, True), (128, 3, 1, 16, 64, True, False), (64, 5, 1, 64, 64, True, True), (64, 4, 3, 16, 6, False, False),
    (96, 3, 3, 48, 96, True, True), (96, 2, 1, 16, 34, False, False), (256, 3, 1, 128, 256, False, True),
    (256, 2, 5, 16, 200, True, False), (256, 1, 1, 16, 0, True, False), (128, 33, 1, 16, 8, True, True)])
@pytest.mark.parametrize("rows,lens", [([801], [801]), ([5, 0, 400, 1, 430], [21, 0, 713, 1, 439])])
def test_append_of_many_rows(fmt, hd, heads, kv_heads, page, rope_dim, halves, bf16, rows, lens):
    """Enough rows for whole tiles at a time, whose sequences begin and end inside tiles."""
    check_append(fmt, hd, heads, kv_heads, page, rope_dim, halves, bf16, rows, lens)


def test_append_of_many_sequences_of_many_rows():
    """More sequences than lanes count at once, empty ones and an impossible one among them."""
    import torch
    rng = np.random.default_rng(15)
    rows = [int(r) for r in rng.integers(0, 40, 150)]
    lens = [r + int(e) for r, e in zip(rows, rng.integers(0, 30, 150))]
    assert sum(rows) > 8 * 150
    hd = 64
    p = Paged(ref.Q8_0, 1, hd, 16, lens)
    x = torch_of(rng.standard_normal((sum(rows), hd)).astype(np.float32))
    back = torch.full((2, sum(rows), hd), 5.0, device="cuda")
    bad = 77
    assert rows[bad] > 0
    wrong = list(lens)
    wrong[bad] = rows[bad] - 1
    for given, message in ((wrong, "22"), (lens, None)):
        b = p.batch(rows, given)

        def both():
            p.cache.append(b, None, 0, 0, 0, 0, x.data_ptr(), hd, x.data_ptr(), hd, 0, 0, 0)
            p.cache.read(b, back[0].data_ptr(), hd, back[1].data_ptr(), hd, 0)

        want = ref.stored(x.cpu().numpy().reshape(-1, 1, hd), ref.Q8_0).astype(np.float32)[:, 0]
        if message:
            assert message in status_of(both)
            at = sum(rows[:bad])
            want[at:at + rows[bad]] = 5.0
        else:
            both()
            assert capi.kernel_status(0) == 0
        np.testing.assert_array_equal(np_of(back)[0], want)
        np.testing.assert_array_equal(np_of(back)[1], want)


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_and_tiles_leave_the_same_bytes(fmt):
    """A prompt at once, and the same in pieces that are stored row by row."""
    import torch
    rng = np.random.default_rng(14)
    hd, kv, n, far = 128, 3, 900, 70
    x = torch_of(rng.standard_normal((n, 2 * kv * hd)).astype(np.float32))
    freq, gain = capi.rope_frequencies(hd, 10000.0)
    f = torch_of(freq)
    rope, stride = capi.Rope(hd, 0, f.data_ptr(), gain), 2 * kv * hd
    pools, backs = [], []
    for steps in ([n], [150] * 6):
        p = Paged(fmt, kv, hd, 64, [far + n], spare=0)
        done = 0
        for r in steps:
            at = x.data_ptr() + done * stride * 4
            p.cache.append(p.batch([r], [far + done + r]), rope, 0, 0, 0, 0, at, stride, at + kv * hd * 4, stride, 0, 0, 0)
            done += r
        pools.append(p.pool)
        back = torch.empty(2, n, kv * hd, device="cuda")
        done = 0
        for r in steps:
            p.cache.read(p.batch([r], [far + done + r]), back[0, done].data_ptr(), kv * hd, back[1, done].data_ptr(), kv * hd, 0)
            done += r
        backs.append(back)
        assert capi.kernel_status(0) == 0
    assert torch.equal(pools[0], pools[1]) and torch.equal(*backs)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("halves", [False, True])
def test_queries_may_be_rotated_in_place(fmt, halves):
    rng = np.random.default_rng(3)
    heads, hd, n = 4, 128, 37
    p = Paged(fmt, 2, hd, 16, [n])
    qkv = rng.standard_normal((n, heads + 4, hd)).astype(np.float32)
    x = torch_of(qkv.reshape(n, -1))
    freq, gain = capi.rope_frequencies(hd, 5e5)
    f = torch_of(freq)
    at, stride = x.data_ptr(), (heads + 4) * hd
    p.cache.append(p.batch([n], [n]), capi.Rope(hd, int(halves), f.data_ptr(), gain), heads, 0, at, stride, at + heads * hd * 4,
                   stride, at + (heads + 2) * hd * 4, stride, at, 0, stride)
    assert capi.kernel_status(0) == 0
    got = np_of(x).reshape(qkv.shape)
    np.testing.assert_array_equal(got[:, :heads], ref.rotate(qkv[:, :heads], np.arange(n), freq, gain, hd, halves))
    np.testing.assert_array_equal(got[:, heads:], qkv[:, heads:])


@pytest.mark.parametrize("fmt", FMTS)
def test_single_tokens_and_a_prompt_leave_the_same_bytes(fmt):
    import torch
    rng = np.random.default_rng(4)
    hd, kv, n, far = 128, 2, 35, 90000
    x = torch_of(rng.standard_normal((n, 2 * kv * hd)).astype(np.float32))
    freq, gain = capi.rope_frequencies(hd, 10000.0)
    f = torch_of(freq)
    rope, stride = capi.Rope(hd, 0, f.data_ptr(), gain), 2 * kv * hd
    pools = []
    for steps in ([n], [1] * n, [3] * 11 + [2]):
        p = Paged(fmt, kv, hd, 64, [far + n], spare=0)
        done = 0
        for r in steps:
            at = x.data_ptr() + done * stride * 4
            p.cache.append(p.batch([r], [far + done + r], single=r == 1), rope, 0, 0, 0, 0, at, stride, at + kv * hd * 4, stride,
                           0, 0, 0)
            done += r
        assert capi.kernel_status(0) == 0
        pools.append(p.pool)
    assert torch.equal(pools[0], pools[1]) and torch.equal(pools[0], pools[2])


@pytest.mark.parametrize("fmt", [ref.Q4_0, ref.Q8_0])
def test_values_that_no_block_holds(fmt):
    """Infinities and NaN make their own block NaN, values past fp16's scales saturate, tiny ones vanish."""
    import torch
    hd = 64
    v = np.ones((5, 1, hd), dtype=np.float32)
    v[0, 0, 3] = np.inf
    v[1, 0, 40] = np.nan
    v[2, 0, :32] = 3e38
    v[3, 0, :32] = 1e-9
    v[4, 0, 5] = -1e30
    p = Paged(fmt, 1, hd, 16, [5])
    x = torch_of(v.reshape(5, hd))
    b = p.batch([5], [5])
    p.cache.append(b, None, 0, 0, 0, 0, x.data_ptr(), hd, x.data_ptr(), hd, 0, 0, 0)
    out = torch.empty(2, 5, hd, device="cuda")
    p.cache.read(b, out[0].data_ptr(), hd, out[1].data_ptr(), hd, 0)
    assert capi.kernel_status(0) == 0
    want = ref.stored(v, fmt).astype(np.float32)[:, 0]
    np.testing.assert_array_equal(np_of(out)[0], want)
    np.testing.assert_array_equal(np_of(out)[1], want)
    assert np.isnan(want[0, :32]).all() and np.isfinite(want[0, 32:]).all() and np.isfinite(want[2:]).all()


@pytest.mark.parametrize("fmt", [ref.Q4_0, ref.Q8_0])
def test_values_that_no_block_holds_among_many_rows(fmt):
    import torch
    hd, n = 128, 807
    v = np.random.default_rng(5).standard_normal((n, 1, hd)).astype(np.float32)
    v[0, 0, 3], v[17, 0, 40], v[31, 0, 127] = np.inf, np.nan, -np.inf
    v[33, 0, :32], v[400, 0, :32], v[806, 0, 5] = 3e38, 1e-9, -1e30
    p = Paged(fmt, 1, hd, 32, [n])
    x = torch_of(v.reshape(n, hd))
    b = p.batch([n], [n])
    p.cache.append(b, None, 0, 0, 0, 0, x.data_ptr(), hd, x.data_ptr(), hd, 0, 0, 0)
    out = torch.empty(2, n, hd, device="cuda")
    p.cache.read(b, out[0].data_ptr(), hd, out[1].data_ptr(), hd, 0)
    assert capi.kernel_status(0) == 0
    want = ref.stored(v, fmt).astype(np.float32)[:, 0]
    np.testing.assert_array_equal(np_of(out)[0], want)
    np.testing.assert_array_equal(np_of(out)[1], want)
    assert int(np.isnan(want).sum()) == 3 * 32


@pytest.mark.parametrize("n", [3, 900])
def test_q8_0_rounds_half_away_from_zero(n):
    """Halves, and the numbers next to them: 0.5 - 2^-25 plus a half is 1 in fp32, and its nearest whole number is 0."""
    import torch
    hd = 64
    v = np.zeros((n, 1, hd), np.float32)
    v[:, 0, 0], v[:, 0, 32] = 127.0, -127.0  # scales of 1
    halves = np.array([0.5, 1.5, 2.5, 62.5, 63.5, 126.5], np.float32)
    below, above = np.nextafter(halves, np.float32(0)), np.nextafter(halves, np.float32(200))
    x = np.concatenate([halves, below, above])
    v[:, 0, 1:19], v[:, 0, 33:51] = x, -x
    want = np.concatenate([halves + 0.5, halves - 0.5, halves + 0.5])
    p = Paged(ref.Q8_0, 1, hd, 16, [n])
    xd = torch_of(v.reshape(n, hd))
    b = p.batch([n], [n])
    p.cache.append(b, None, 0, 0, 0, 0, xd.data_ptr(), hd, xd.data_ptr(), hd, 0, 0, 0)
    out = torch.empty(2, n, hd, device="cuda")
    p.cache.read(b, out[0].data_ptr(), hd, out[1].data_ptr(), hd, 0)
    assert capi.kernel_status(0) == 0
    for o in np_of(out):
        np.testing.assert_array_equal(o[:, 1:19], np.tile(want, (n, 1)))
        np.testing.assert_array_equal(o[:, 33:51], np.tile(-want, (n, 1)))


# ---- attention -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,heads,kv_heads,page", [(128, 8, 1, 64), (128, 4, 4, 16), (64, 14, 2, 32), (96, 9, 3, 16),
                                                    (256, 4, 2, 128), (128, 24, 1, 16)])
def test_single_tokens(fmt, hd, heads, kv_heads, page):
    lens = [1, 16, 17, 700, 2, 333]
    p = Paged(fmt, kv_heads, hd, page, lens, seed=hd)
    check_attention(p, [1] * 6, lens, heads, np.random.default_rng(hd + heads), single=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,lens", [([3, 5, 1], [3, 70, 1]), ([9], [2500]), ([2, 0, 4], [31, 12, 64]), ([33], [33])])
@pytest.mark.parametrize("window", [0, 1, 20])
def test_several_rows_and_windows(fmt, rows, lens, window):
    p = Paged(fmt, 2, 128, 32, lens, seed=len(rows))
    check_attention(p, rows, lens, 6, np.random.default_rng(sum(lens)), window=window)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("bf16,out_bf16", [(True, False), (False, True), (True, True)])
def test_types_of_rows(fmt, bf16, out_bf16):
    lens = [100, 37]
    p = Paged(fmt, 2, 128, 16, lens)
    check_attention(p, [2, 3], lens, 8, np.random.default_rng(9), bf16, out_bf16)


def test_many_sequences_of_few_tokens():
    """More sequences than a CTA has threads: the list of tiles is found in several rounds."""
    lens = [1 + i % 23 for i in range(300)]
    p = Paged(ref.Q4_0, 1, 64, 16, lens)
    check_attention(p, [1] * 300, lens, 2, np.random.default_rng(1), single=True)


@pytest.mark.parametrize("fmt", FMTS)
def test_one_long_sequence_among_short_ones(fmt):
    lens = [5, 9000, 1, 40]
    p = Paged(fmt, 1, 128, 64, lens)
    check_attention(p, [1] * 4, lens, 8, np.random.default_rng(2), single=True)


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_that_see_nothing_give_zeros(fmt):
    """A sequence of length zero, and rows in front of a sequence's first token."""
    rng = np.random.default_rng(5)
    p = Paged(fmt, 1, 64, 16, [0, 3, 20])
    ks, vs = p.fill(rng)
    rows, lens = [2, 5, 1], [0, 3, 20]
    q = rng.standard_normal((8, 2, 64)).astype(np.float32)
    got = p.attend(q, rows, lens, 2)
    want = np.concatenate([ref.attention(q[a:a + r], ks[s], vs[s], n, 0.125) for s, (a, r, n) in
                           enumerate(zip([0, 2, 7], rows, lens))])
    assert (got[:4] == 0).all()
    np.testing.assert_allclose(got, want, atol=ref.attention_bound(q, ks[2], vs[2], 0.125, False) +
                               ref.attention_bound(q, ks[1], vs[1], 0.125, False), rtol=0)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows", [1, 6])
def test_what_a_row_does_not_see_does_not_reach_it(fmt, rows):
    """NaN in a later token, in front of the window, behind the length: only the rows that see them."""
    rng = np.random.default_rng(6)
    n, hd, heads = 45, 128, 4
    p = Paged(fmt, 1, hd, 16, [n])
    k = rng.standard_normal((n, 1, hd)).astype(np.float32)
    v = rng.standard_normal((n, 1, hd)).astype(np.float32)
    for bad in (np.nan, np.inf):
        v2, k2 = v.copy(), k.copy()
        v2[n - 3, 0, 70] = bad     # token n - 3 is seen by the last three rows
        k2[4, 0, 7] = np.nan       # in front of the window
        v2[5, 0, 7] = bad
        kd, vd = torch_of(k2), torch_of(v2)
        p.cache.append(p.batch([n], [n]), None, 0, 0, 0, 0, kd.data_ptr(), hd, vd.data_ptr(), hd, 0, 0, 0)
        q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
        got = p.attend(q, [rows], [n], heads, window=30)
        sees = np.arange(n - rows, n) >= n - 3
        assert np.isfinite(got[~sees]).all()
        touched = [70] if fmt == ref.F16 else range(64, 96)
        assert not np.isfinite(got[sees][:, :, touched]).any()
        others = np.setdiff1d(np.arange(hd), touched)
        kk, vv = ref.stored(k2, fmt), ref.stored(v2, fmt)
        want = ref.attention(q, np.nan_to_num(kk), np.where(np.isfinite(vv), vv, 0), n, hd ** -0.5, 30)
        bound = ref.attention_bound(q, np.nan_to_num(kk), np.where(np.isfinite(vv), vv, 0), hd ** -0.5, False)
        assert np.abs(got - want)[:, :, others].max() <= bound
        if (~sees).any():
            assert np.abs(got - want)[~sees].max() <= bound


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("size", [1.0, 1e-2])
def test_a_token_of_nan_leaves_other_rows_their_precision(fmt, size):
    """The first tile that the call sees holds one token that the first row alone sees, and nothing of its value is a number."""
    rng = np.random.default_rng(35)
    n, hd, heads, rows, window = 213, 64, 4, 3, 100
    p = Paged(fmt, 1, hd, 16, [n])
    k = rng.standard_normal((n, 1, hd)).astype(np.float32)
    v = (rng.standard_normal((n, 1, hd)) * size).astype(np.float32)
    first = n - rows - window + 1
    assert first % 16 == 15
    v[first] = np.nan
    kd, vd = torch_of(k), torch_of(v)
    p.cache.append(p.batch([n], [n]), None, 0, 0, 0, 0, kd.data_ptr(), hd, vd.data_ptr(), hd, 0, 0, 0)
    q = (rng.standard_normal((rows, heads, hd)) * 2).astype(np.float32)
    got = p.attend(q, [rows], [n], heads, window=window)
    want = ref.attention(q, ref.stored(k, fmt), ref.stored(v, fmt), n, hd ** -0.5, window)
    assert np.isnan(got[0]).all() and np.isnan(want[0]).all()
    assert np.linalg.norm(got[1:] - want[1:]) <= np.linalg.norm(want[1:]) * ref.fp32_norm_bound(2.0)


def test_a_row_of_nothing_but_nan_is_nan():
    rng = np.random.default_rng(7)
    p = Paged(ref.Q4_0, 1, 64, 16, [700, 10])
    p.fill(rng)
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    q[0, 1, 5] = np.nan
    got = p.attend(q, [1, 1], [700, 10], 4, single=True)
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[0, [0, 2, 3]]).all() and np.isfinite(got[1]).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_large_and_small_magnitudes(fmt):
    """Scores of a hundred, values of 1e-4 beside values of 1e3, queries of 1e-6 and 1e6."""
    rng = np.random.default_rng(8)
    n, hd = 600, 64
    p = Paged(fmt, 1, hd, 16, [n])
    k = rng.standard_normal((n, 1, hd)).astype(np.float32) * 4
    v = (rng.standard_normal((n, 1, hd)) * 10.0 ** rng.integers(-4, 4, (n, 1, 1))).astype(np.float32)
    kd, vd = torch_of(k), torch_of(v)
    p.cache.append(p.batch([n], [n]), None, 0, 0, 0, 0, kd.data_ptr(), hd, vd.data_ptr(), hd, 0, 0, 0)
    kk, vv = ref.stored(k, fmt), ref.stored(v, fmt)
    for size in (1e-6, 1.0, 8.0):
        q = rng.standard_normal((1, 3, hd)).astype(np.float32) * np.float32(size)
        got = p.attend(q, [1], [n], 3)
        want = ref.attention(q, kk, vv, n, hd ** -0.5)
        assert np.abs(got - want).max() <= ref.attention_bound(q, kk, vv, hd ** -0.5, False)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("size", [100.0, 1.0, 1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("hd,heads,n", [(64, 4, 20), (64, 32, 700), (128, 4, 500), (128, 24, 2500), (96, 4, 333), (256, 4, 90)])
def test_fp32_results_carry_fp32_s_precision(fmt, size, hd, heads, n):
    """In the 2-norm, whatever the size of the values: scales of blocks down to fp16's smallest."""
    rng = np.random.default_rng(32)
    p = Paged(fmt, 1, hd, 16, [n])
    k = rng.standard_normal((n, 1, hd)).astype(np.float32)
    v = (rng.standard_normal((n, 1, hd)) * size).astype(np.float32)
    kd, vd = torch_of(k), torch_of(v)
    p.cache.append(p.batch([n], [n]), None, 0, 0, 0, 0, kd.data_ptr(), hd, vd.data_ptr(), hd, 0, 0, 0)
    q = (rng.standard_normal((3, heads, hd)) * 2).astype(np.float32)
    got = p.attend(q, [3], [n], heads)
    want = ref.attention(q, ref.stored(k, fmt), ref.stored(v, fmt), n, hd ** -0.5)
    assert np.linalg.norm(want) > 0 and np.linalg.norm(got - want) <= np.linalg.norm(want) * ref.fp32_norm_bound(2.0)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e6, 1e8, 1e20])
def test_scores_of_any_size(fmt, prompt, size):
    """One key takes all: scores past 2^24, whose last bits are whole powers of two of a probability."""
    rng = np.random.default_rng(37)
    n, rows, heads, hd = 300, 150, 4, 64
    p = Paged(fmt, 1, hd, 16, [n])
    k = (rng.standard_normal((n, 1, hd)) * np.linspace(0.5, 2, n)[:, None, None]).astype(np.float32)  # maxima come late, too
    v = rng.standard_normal((n, 1, hd)).astype(np.float32)
    kd, vd = torch_of(k), torch_of(v)
    p.cache.append(p.batch([n], [n]), None, 0, 0, 0, 0, kd.data_ptr(), hd, vd.data_ptr(), hd, 0, 0, 0)
    kk, vv = ref.stored(k, fmt)[:, 0], ref.stored(v, fmt)[:, 0]
    q = (rng.standard_normal((rows, heads, hd)) * size).astype(np.float32)
    got = p.attend(q, [rows], [n], heads, out_bf16=prompt, prompt=prompt)
    score = np.einsum("rhd,nd->rhn", q.astype(np.float64), kk) * hd ** -0.5
    score[np.arange(n)[None, None] > (n - rows + np.arange(rows))[:, None, None] + np.zeros((1, heads, 1))] = -np.inf
    first, second = np.sort(score, -1)[..., -1], np.sort(score, -1)[..., -2]
    # with fp16 operands (the prompt kernel's) each product is off by up to 2^-10 of itself, for two keys of at most 16: 2^-5 of q's
    # magnitudes; and e^-40 is nothing
    assert np.abs(kk).max() < 16
    clear = (first - second > 2.0 ** -5 * np.abs(q).sum(-1) * hd ** -0.5) & (first - second > 40)
    assert clear.mean() > 0.5 or size < 1e4
    want = vv[score.argmax(-1)]
    assert np.isfinite(got).all()
    bound = np.abs(want) * (2.0 ** -8 + 2.0 ** -10 if prompt else 2.0 ** -20) + 1e-15
    assert (np.abs(got - want) <= bound)[clear].all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0, 1e-20])
def test_scales_of_any_sign_and_size(fmt, prompt, scale):
    """0 and 1e-20: the mean of what a row sees."""
    rng = np.random.default_rng(38)
    n, rows, heads, hd = 200, 130, 4, 64
    p = Paged(fmt, 2, hd, 16, [n])
    ks, vs = p.fill(rng)
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    got = p.attend(q, [rows], [n], heads, out_bf16=prompt, prompt=prompt, scale=scale, window=150)
    want = ref.attention(q, ks[0], vs[0], n, np.float64(np.float32(scale)), 150)
    size = abs(scale) * hd ** 0.5  # of the scores
    bound = 2.0 ** -8 + 4 * 2.0 ** -11 * (size + 1) if prompt else ref.fp32_norm_bound(size)
    assert np.linalg.norm(got - want) <= np.linalg.norm(want) * bound


def test_padding_rows_and_strided_rows_stay_as_they_were():
    import torch
    rng = np.random.default_rng(11)
    p = Paged(ref.Q8_0, 2, 64, 16, [50, 9])
    ks, vs = p.fill(rng)
    rows, lens, heads, wide = [3, 1], [50, 9], 4, 4 * 64 + 24
    q = rng.standard_normal((7, wide)).astype(np.float32)
    qd = torch_of(q)
    out = torch.full((7, wide), 5.0, device="cuda")
    p.cache.attend(p.batch(rows, lens, total=7), heads, qd.data_ptr() + 32, 0, wide, out.data_ptr() + 64, 0, wide, 0.125, 0,
                   p.workspace.data_ptr())
    assert capi.kernel_status(0) == 0
    o = np_of(out)
    assert (o[4:] == 5.0).all() and (o[:, :16] == 5.0).all() and (o[:, 16 + 256:] == 5.0).all()
    qq = q[:, 8:8 + 256].reshape(7, heads, 64)
    want = np.concatenate([ref.attention(qq[:3], ks[0], vs[0], 50, 0.125), ref.attention(qq[3:4], ks[1], vs[1], 9, 0.125)])
    assert np.abs(o[:4, 16:16 + 256].reshape(4, heads, 64) - want).max() <= ref.attention_bound(qq, ks[0], vs[0], 0.125, False)


def test_same_inputs_same_bits_and_a_clean_workspace():
    import torch
    rng = np.random.default_rng(12)
    lens = [3000, 800, 5]
    p = Paged(ref.Q4_0, 2, 128, 64, lens)
    p.fill(rng)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    first = p.attend(q, [1] * 3, lens, 8, single=True)
    for _ in range(3):
        np.testing.assert_array_equal(p.attend(q, [1] * 3, lens, 8, single=True), first)
    # the first 16 KiB hold the counters that a call leaves zeroed
    assert int(p.workspace[:16384].to(torch.int32).sum()) == 0


def test_replayed_graph_follows_the_lengths():
    """append + attend captured once: each replay appends one token more, on a stream of its own."""
    import torch
    rng = np.random.default_rng(13)
    hd, heads, kv, n, steps = 128, 8, 2, 40, 6
    p = Paged(ref.Q4_0, kv, hd, 16, [n + steps, 20 + steps])
    full = rng.standard_normal((2, n + steps, 2 * kv, hd)).astype(np.float32)
    freq, gain = capi.rope_frequencies(hd, 10000.0)
    f = torch_of(freq)
    rope = capi.Rope(hd, 0, f.data_ptr(), gain)
    stride = (heads + 2 * kv) * hd
    for s, m in enumerate([n, 20]):  # the prompts
        x = torch_of(full[s, :m].reshape(m, -1))
        b = p.batch([m], [m])
        b.page_table_dev = p.table_dev[s].data_ptr()
        p.cache.append(b, rope, 0, 0, 0, 0, x.data_ptr(), 2 * kv * hd, x.data_ptr() + kv * hd * 4, 2 * kv * hd, 0, 0, 0)
    qkv = torch.zeros(2, stride, device="cuda")
    length = torch.tensor([n, 20], device="cuda", dtype=torch.int32)
    out = torch.zeros(2, heads * hd, device="cuda")
    b = capi.KVBatch(2, p.width, p.table_dev.data_ptr(), length.data_ptr(), 0, 2)
    at = qkv.data_ptr()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()

    def step():
        length.add_(1)
        p.cache.append(b, rope, heads, 0, at, stride, at + heads * hd * 4, stride, at + (heads + kv) * hd * 4, stride, at, 0,
                       stride, stream.cuda_stream)
        p.cache.attend(b, heads, at, 0, stride, out.data_ptr(), 0, heads * hd, hd ** -0.5, 0, p.workspace.data_ptr(),
                       stream.cuda_stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            step()
    length.copy_(torch.tensor([n, 20]))
    for i in range(steps):
        q = rng.standard_normal((2, heads, hd)).astype(np.float32)
        new = np.stack([full[0, n + i], full[1, 20 + i]])
        torch.cuda.synchronize()
        qkv.copy_(torch_of(np.concatenate([q, new], 1).reshape(2, -1)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = np_of(out).reshape(2, heads, hd)
        for s, m in enumerate([n + i + 1, 20 + i + 1]):
            pos = np.arange(m)
            keys = ref.stored(ref.rotate(full[s, :m, :kv], pos, freq, gain, hd, False), ref.Q4_0)
            vals = ref.stored(full[s, :m, kv:], ref.Q4_0)
            qr = ref.rotate(q[s:s + 1], pos[-1:], freq, gain, hd, False)
            want = ref.attention(qr, keys, vals, m, hd ** -0.5)
            assert np.abs(got[s] - want[0]).max() <= ref.attention_bound(qr, keys, vals, hd ** -0.5, False)
    assert capi.kernel_status(0) == 0
    del graph


def test_two_calls_at_once_on_two_streams():
    import torch
    rng = np.random.default_rng(14)
    caches = [Paged(ref.Q4_0, 2, 128, 64, [5000, 77], seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in caches]
    data = [(p.fill(rng), rng.standard_normal((2, 8, 128)).astype(np.float32)) for p in caches]
    qs = [torch_of(q.reshape(2, -1)) for _, q in data]
    outs = [torch.zeros(2, 8 * 128, device="cuda") for _ in caches]
    batches = [p.batch([1, 1], [5000, 77], single=True) for p in caches]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, s, q, o, b in zip(caches, streams, qs, outs, batches):
            p.cache.attend(b, 8, q.data_ptr(), 0, 1024, o.data_ptr(), 0, 1024, 128 ** -0.5, 0, p.workspace.data_ptr(),
                           s.cuda_stream)
    torch.cuda.synchronize()
    assert capi.kernel_status(0) == 0
    for ((ks, vs), q), o in zip(data, outs):
        for s, n in enumerate([5000, 77]):
            want = ref.attention(q[s:s + 1], ks[s], vs[s], n, 128 ** -0.5)
            assert np.abs(np_of(o)[s].reshape(8, 128) - want[0]).max() <= ref.attention_bound(q[s:s + 1], ks[s], vs[s],
                                                                                              128 ** -0.5, False)


def test_pool_past_32_bits():
    """The last pages of a pool of more than 4 GiB."""
    import torch
    rng = np.random.default_rng(15)
    hd, kv, page = 128, 8, 128
    per_page = capi.kv_pool_bytes(ref.F16, kv, hd, page, 1)
    n_pages = (5 << 30) // per_page
    pool = torch.empty(n_pages * per_page, dtype=torch.uint8, device="cuda")
    cache = capi.KVCache(ref.F16, kv, hd, page, n_pages, pool.data_ptr())
    n = 200
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device="cuda")
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    begin = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    k, v = rng.standard_normal((2, n, kv, hd)).astype(np.float32)
    kd, vd = torch_of(k), torch_of(v)
    cache.append(capi.KVBatch(1, 2, table.data_ptr(), length.data_ptr(), begin.data_ptr(), n), None, 0, 0, 0, 0, kd.data_ptr(),
                 kv * hd, vd.data_ptr(), kv * hd, 0, 0, 0)
    q = rng.standard_normal((1, kv, hd)).astype(np.float32)
    qd = torch_of(q)
    out = torch.empty(1, kv * hd, device="cuda")
    work = torch.zeros(capi.KV_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    cache.attend(capi.KVBatch(1, 2, table.data_ptr(), length.data_ptr(), 0, 1), kv, qd.data_ptr(), 0, kv * hd, out.data_ptr(), 0,
                 kv * hd, hd ** -0.5, 0, work.data_ptr())
    assert capi.kernel_status(0) == 0
    kk, vv = ref.stored(k, ref.F16), ref.stored(v, ref.F16)
    want = ref.attention(q, kk, vv, n, hd ** -0.5)
    assert np.abs(np_of(out).reshape(1, kv, hd) - want).max() <= ref.attention_bound(q, kk, vv, hd ** -0.5, False)


# ---- prompts: the tensor cores' 128-column tiles -----------------------------------------------------------------------------

def check_prompt(p, rows, lens, heads, rng, bf16=False, window=0, q_scale=2.0, poison=()):
    """bf16 results against 64 bits, element by element and in the 2-norm."""
    ks, vs = p.fill(rng)
    q = (rng.standard_normal((sum(rows), heads, p.hd)) * q_scale).astype(np.float32)
    if bf16:
        q = ref.bf16_round(q)
    got = p.attend(q, rows, lens, heads, bf16, True, window, prompt=True)
    at, off, size = 0, 0.0, 0.0
    for s, (n, r) in enumerate(zip(lens, rows)):
        if r == 0:
            continue
        want = ref.attention(q[at:at + r], ks[s], vs[s], n, p.hd ** -0.5, window)
        err = np.abs(got[at:at + r] - want)
        assert err.max() <= ref.attention_bound(q[at:at + r], ks[s], vs[s], p.hd ** -0.5, True, True), (s, err.max())
        off, size = off + (err ** 2).sum(), size + (want ** 2).sum()
        at += r
    assert off <= size * ref.norm_bound(p.hd, q_scale, 1.0, True) ** 2, (off / size) ** 0.5


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,heads,kv_heads,page", [(128, 2, 2, 64), (64, 8, 2, 16), (128, 7, 1, 32)])
@pytest.mark.parametrize("rows,lens", [([256], [256]), ([130, 1, 0, 67], [130, 40, 9, 300]), ([100], [1000]), ([300], [301])])
def test_prompts(fmt, hd, heads, kv_heads, page, rows, lens):
    p = Paged(fmt, kv_heads, hd, page, lens, seed=sum(rows))
    check_prompt(p, rows, lens, heads, np.random.default_rng(hd + sum(lens)), bf16=heads == 7)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window", [1, 17, 200])
def test_prompts_with_windows(fmt, window):
    p = Paged(fmt, 1, 128, 16, [500, 90])
    check_prompt(p, [333, 90], [500, 90], 2, np.random.default_rng(window), window=window)


def test_prompts_of_more_items_than_sms():
    lens = [64 + 3 * i for i in range(90)]
    p = Paged(ref.Q4_0, 2, 64, 16, lens)
    check_prompt(p, [64] * 90, lens, 4, np.random.default_rng(20))


def test_prompts_whose_scores_grow_along_the_keys():
    """The running maximum moves by more than its slack again and again."""
    rng = np.random.default_rng(21)
    n, hd = 700, 128
    p = Paged(ref.F16, 1, hd, 64, [n])
    k = rng.standard_normal((n, 1, hd)).astype(np.float32) * np.linspace(0.05, 4, n)[:, None, None].astype(np.float32)
    v = rng.standard_normal((n, 1, hd)).astype(np.float32)
    kd, vd = torch_of(k), torch_of(v)
    p.cache.append(p.batch([n], [n]), None, 0, 0, 0, 0, kd.data_ptr(), hd, vd.data_ptr(), hd, 0, 0, 0)
    q = rng.standard_normal((128, 2, hd)).astype(np.float32) * 4
    got = p.attend(q, [128], [n], 2, out_bf16=True, prompt=True)
    kk, vv = ref.stored(k, ref.F16), ref.stored(v, ref.F16)
    want = ref.attention(q, kk, vv, n, hd ** -0.5)
    assert np.linalg.norm(got - want) <= np.linalg.norm(want) * ref.norm_bound(hd, 4.0, 4.0, True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,below,sink_value", [(3000, 10.0, 0.0), (3000, 20.6, 0.0), (3000, 24.4, 0.0), (40000, 20.4, 0.01), (40000, 24.4, 0.01)])
@pytest.mark.parametrize("last", [False, True])
def test_prompts_with_a_long_tail_below_one_key(fmt, n, below, sink_value, last):
    """One key that takes nearly all of the probability and has hardly a value, before or behind many that are alike."""
    rng = np.random.default_rng(33)
    hd, heads, rows = 64, 2, 150
    p = Paged(fmt, 1, hd, 16, [n])
    k = np.zeros((n, 1, hd), np.float32)
    v = (np.abs(rng.standard_normal((n, 1, hd))) + 0.5).astype(np.float32)
    at = n - rows if last else 0
    k[at], v[at] = 1.0, sink_value
    kd, vd = torch_of(k), torch_of(v)
    p.cache.append(p.batch([n], [n]), None, 0, 0, 0, 0, kd.data_ptr(), hd, vd.data_ptr(), hd, 0, 0, 0)
    kk, vv = ref.stored(k, fmt)[:, 0], ref.stored(v, fmt)[:, 0]
    scale = np.float32(below * np.log(2) / kk[at].sum())  # queries of ones
    got = p.attend(np.ones((rows, heads, hd), np.float32), [rows], [n], heads, out_bf16=True, prompt=True, scale=float(scale))
    w = np.exp2(np.float64(scale) * kk.sum(-1) / np.log(2) - below)[:, None]
    total, mass = np.cumsum(w, 0)[n - rows:], np.cumsum(w * vv, 0)[n - rows:]
    want = (mass / total)[:, None]
    # bf16's half step; fp16 of a probability and of a value; half of fp16's last bit, 2^-32.75 of the largest, for every key.  A
    # maximum behind the tail scales the sums that were there down, in fp32
    bound = want * (2.0 ** -8 + 2 * 2.0 ** -11 + 2.0 ** -18) + n * 2.0 ** -32.75 * vv.max()
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / want).max()


@pytest.mark.parametrize("fmt", FMTS)
def test_prompts_what_a_row_does_not_see_does_not_reach_it(fmt):
    rng = np.random.default_rng(22)
    n, rows, hd, heads = 400, 200, 128, 2
    p = Paged(fmt, 1, hd, 16, [n])
    k = rng.standard_normal((n, 1, hd)).astype(np.float32)
    v = rng.standard_normal((n, 1, hd)).astype(np.float32)
    k[250, 0, 3], v[330, 0, 70], v[20, 0, 1] = np.nan, np.inf, np.nan  # token 20 lies in front of every window
    kd, vd = torch_of(k), torch_of(v)
    p.cache.append(p.batch([n], [n]), None, 0, 0, 0, 0, kd.data_ptr(), hd, vd.data_ptr(), hd, 0, 0, 0)
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    got = p.attend(q, [rows], [n], heads, out_bf16=True, prompt=True, window=100)
    pos = np.arange(n - rows, n)
    sees = ((pos >= 250) & (pos < 350)) | (pos >= 330)
    assert np.isfinite(got[~sees]).all() and not np.isfinite(got[sees][:, :, 70]).any()
    kk, vv = np.nan_to_num(ref.stored(k, fmt)), ref.stored(v, fmt)
    vv = np.where(np.isfinite(vv), vv, 0)
    want = ref.attention(q, kk, vv, n, hd ** -0.5, 100)[~sees]
    assert np.linalg.norm(got[~sees] - want) <= np.linalg.norm(want) * ref.norm_bound(hd, 1.0, 1.0, True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,window", [(128, 100), (64, 0)])
def test_prompts_a_value_that_is_not_finite_stays_in_its_dimension(fmt, hd, window):
    """Quants: in its block of 32.  The other dimensions of the rows that see it are what they are without it."""
    rng = np.random.default_rng(34)
    n, rows, heads = 400, 200, 2
    p = Paged(fmt, 1, hd, 16, [n])
    k = rng.standard_normal((n, 1, hd)).astype(np.float32)
    v = rng.standard_normal((n, 1, hd)).astype(np.float32)
    v[330, 0, hd - 58], v[20, 0, 1], v[399, 0, hd - 1], v[210, 0, 0], v[331, 0, 33] = np.inf, np.nan, -np.inf, np.nan, np.inf
    if window == 0:
        v[20, 0, 1], v[210, 0, 0] = 0.0, 0.0  # every row would see them
    kd, vd = torch_of(k), torch_of(v)
    p.cache.append(p.batch([n], [n]), None, 0, 0, 0, 0, kd.data_ptr(), hd, vd.data_ptr(), hd, 0, 0, 0)
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    got = p.attend(q, [rows], [n], heads, out_bf16=True, prompt=True, window=window)
    kk, vv = ref.stored(k, fmt), ref.stored(v, fmt)
    odd = ~np.isfinite(ref.attention(q, kk, vv, n, hd ** -0.5, window))
    assert odd.any() and not odd.all()
    np.testing.assert_array_equal(~np.isfinite(got), odd)
    want = ref.attention(q, kk, np.where(np.isfinite(vv), vv, 0), n, hd ** -0.5, window)
    assert np.linalg.norm((got - want)[~odd]) <= np.linalg.norm(want[~odd]) * ref.norm_bound(hd, 1.0, 1.0, True)


@pytest.mark.parametrize("fmt", FMTS)
def test_prompts_rows_that_see_nothing_and_padding(fmt):
    rng = np.random.default_rng(23)
    p = Paged(fmt, 1, 64, 16, [30, 0])
    ks, vs = p.fill(rng)
    q = rng.standard_normal((250, 2, 64)).astype(np.float32)
    got = p.attend(q, [130, 70], [30, 0], 2, out_bf16=True, prompt=True, total=250)
    assert (got[:100] == 0).all() and (got[130:200] == 0).all() and (got[200:] == 7).all()
    want = ref.attention(q[100:130], ks[0], vs[0], 30, 0.125)
    assert np.linalg.norm(got[100:130] - want) <= np.linalg.norm(want) * ref.norm_bound(64, 1.0, 1.0, True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 4, 2 ** 30])
@pytest.mark.parametrize("prompt", [False, True])
def test_a_window_wider_than_any_sequence_is_none(fmt, window, prompt):
    """With rows in front of the first token, in either kernel: the bits of a call without a window."""
    rng = np.random.default_rng(31)
    p = Paged(fmt, 1, 64, 16, [30, 3])
    p.fill(rng)
    q = rng.standard_normal((160, 4, 64)).astype(np.float32)
    got = [p.attend(q, [150, 10], [30, 3], 4, out_bf16=prompt, prompt=prompt, window=w) for w in (0, window)]
    sees = np.r_[120:150, 157:160]
    assert got[0][sees].any(-1).all() and not np.delete(got[0], sees, 0).any()
    np.testing.assert_array_equal(got[1], got[0])


def test_prompts_repeat_bit_for_bit_and_leave_the_workspace_clean():
    rng = np.random.default_rng(24)
    import torch
    p = Paged(ref.Q4_0, 4, 64, 16, [600, 200])
    p.fill(rng)
    q = rng.standard_normal((700, 8, 64)).astype(np.float32)
    first = p.attend(q, [500, 200], [600, 200], 8, out_bf16=True, prompt=True)
    for _ in range(3):
        np.testing.assert_array_equal(p.attend(q, [500, 200], [600, 200], 8, out_bf16=True, prompt=True), first)
    assert int(p.workspace[:16384].to(torch.int32).sum()) == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_prompts_captured_once_follow_rows_and_lengths(fmt):
    """Tiles appended and prompts attended in one graph, whose rows are cut differently at every replay."""
    import torch
    rng = np.random.default_rng(27)
    hd, heads, kv, total = 64, 4, 2, 1024
    p = Paged(fmt, kv, hd, 32, [total] * 3)
    width = heads + 2 * kv
    qkv = rng.standard_normal((total, width, hd)).astype(np.float32)
    x, freq = torch_of(qkv.reshape(total, -1)), capi.rope_frequencies(hd, 10000.0)[0]
    f = torch_of(freq)
    rope, stride = capi.Rope(hd, 1, f.data_ptr(), 1.0), width * hd
    q = torch.zeros(total, heads * hd, device="cuda")
    out = torch.zeros(total, heads * hd, device="cuda", dtype=torch.bfloat16)
    begin, length = (torch.zeros(n, device="cuda", dtype=torch.int32) for n in (4, 3))
    b = capi.KVBatch(3, p.width, p.table_dev.data_ptr(), length.data_ptr(), begin.data_ptr(), total)
    stream, at = torch.cuda.Stream(), x.data_ptr()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            p.cache.append(b, rope, heads, 0, at, stride, at + heads * hd * 4, stride, at + (heads + kv) * hd * 4, stride,
                           q.data_ptr(), 0, heads * hd, stream.cuda_stream)
            p.cache.attend(b, heads, q.data_ptr(), 0, heads * hd, out.data_ptr(), 1, heads * hd, 0.125, 0,
                           p.workspace.data_ptr(), stream.cuda_stream)
    for rows in ([300, 0, 200], [1, 700, 300], [0, 0, 0], [513, 31, 33]):
        cut = np.concatenate([[0], np.cumsum(rows)])
        begin.copy_(torch_of(cut.astype(np.int32)))
        length.copy_(torch_of(np.asarray(rows, dtype=np.int32)))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = np_of(out).reshape(total, heads, hd)
        assert (got[cut[-1]:] == 7.0).all()
        for s, n in enumerate(rows):
            if n:
                part = qkv[cut[s]:cut[s + 1]]
                turned = ref.rotate(part[:, :heads + kv], np.arange(n), freq, 1.0, hd, True)
                keys, vals = ref.stored(turned[:, heads:], fmt), ref.stored(part[:, heads + kv:], fmt)
                want = ref.attention(turned[:, :heads], keys, vals, n, 0.125)
                assert np.abs(got[cut[s]:cut[s + 1]] - want).max() <= ref.attention_bound(turned[:, :heads], keys, vals, 0.125,
                                                                                          True, True)
    assert capi.kernel_status(0) == 0
    del graph


def test_prompts_queries_that_are_not_finite_stay_their_own_rows():
    rng = np.random.default_rng(28)
    n, rows, heads, hd = 300, 150, 2, 128
    p = Paged(ref.Q4_0, 1, hd, 16, [n])
    ks, vs = p.fill(rng)
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    q[3, 1, 5], q[140, 0, 127] = np.nan, np.inf
    got = p.attend(q, [rows], [n], heads, out_bf16=True, prompt=True)
    odd = np.zeros((rows, heads), dtype=bool)
    odd[3, 1] = odd[140, 0] = True
    assert np.isnan(got[odd]).all() and np.isfinite(got[~odd]).all()
    want = ref.attention(np.nan_to_num(q, posinf=0.0), ks[0], vs[0], n, hd ** -0.5)
    assert np.linalg.norm((got - want)[~odd]) <= np.linalg.norm(want) * ref.norm_bound(hd, 1.0, 1.0, True)


def test_prompts_bad_pages_and_rows():
    rng = np.random.default_rng(25)
    import torch
    p = Paged(ref.Q4_0, 1, 64, 16, [200, 200])
    ks, vs = p.fill(rng)
    good = p.table_dev.clone()
    q = rng.standard_normal((200, 2, 64)).astype(np.float32)
    qd, out = torch.zeros(2048, 128, device="cuda"), torch.zeros(2048, 128, device="cuda", dtype=torch.bfloat16)
    qd[:200] = torch_of(q.reshape(200, -1))

    def attend(b):
        p.cache.attend(b, 2, qd.data_ptr(), 0, 128, out.data_ptr(), 1, 128, 0.125, 0, p.workspace.data_ptr())

    for page in (-1, p.n_pages):
        p.table_dev[0, 5] = page
        assert "21" in status_of(lambda: attend(p.batch([100, 100], [200, 200], total=2048)))
        want = ref.attention(q[100:], ks[1], vs[1], 200, 0.125)
        assert np.linalg.norm(np_of(out)[100:200].reshape(100, 2, 64) - want) <= np.linalg.norm(want) * ref.norm_bound(64, 1.0, 1.0, True)
    p.table_dev.copy_(good)
    assert "22" in status_of(lambda: attend(p.batch([100, 100], [p.width * 16 + 1, 200], total=2048)))
    assert "22" in status_of(lambda: attend(p.batch([100, 1949], [200, 2000], total=2048)))
    assert int(p.workspace[:16384].to(torch.int32).sum()) == 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("appended", [300, 900])
def test_the_last_positions_that_a_table_can_name(fmt, appended):
    """Positions near 2^31: appended row by row or in tiles, attended by few rows and by a prompt, with a window."""
    import torch
    rng = np.random.default_rng(36)
    hd, heads, page, width, window = 64, 4, 65536, 32766, 100
    n = width * page - 20
    pool = torch.zeros(capi.kv_pool_bytes(fmt, 1, hd, page, 1), dtype=torch.uint8, device="cuda")
    cache = capi.KVCache(fmt, 1, hd, page, 1, pool.data_ptr())
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")  # one page holds what is looked at
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    work = torch.zeros(capi.KV_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")

    def batch(rows, total=None):
        begin = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        return capi.KVBatch(1, width, table.data_ptr(), length.data_ptr(), begin.data_ptr(), total or rows), begin

    x = rng.standard_normal((appended, heads + 2, hd)).astype(np.float32)
    xd, q_out = torch_of(x.reshape(appended, -1)), torch.zeros(appended, heads * hd, device="cuda")
    freq, gain = capi.rope_frequencies(hd, 10000.0)
    f = torch_of(freq)
    at, stride = xd.data_ptr(), (heads + 2) * hd
    b, hold = batch(appended)
    cache.append(b, capi.Rope(hd, 0, f.data_ptr(), gain), heads, 0, at, stride, at + heads * hd * 4, stride, at + (heads + 1) * hd * 4,
                 stride, q_out.data_ptr(), 0, heads * hd)
    back = torch.zeros(2, appended, hd, device="cuda")
    cache.read(b, back[0].data_ptr(), hd, back[1].data_ptr(), hd, 0)
    assert capi.kernel_status(0) == 0
    pos = np.arange(n - appended, n)
    turned = ref.rotate(x[:, :heads + 1], pos, freq, gain, hd, False)
    # both sides take the sine and the cosine of the same 64-bit angle: the results are the same but for fp32's last bit
    np.testing.assert_allclose(np_of(q_out).reshape(appended, heads, hd), turned[:, :heads], rtol=2.0 ** -22, atol=2.0 ** -40)
    np.testing.assert_array_equal(np_of(back)[1], ref.stored(x[:, heads + 1], fmt).astype(np.float32))
    keys, vals = np_of(back)[0][:, None].astype(np.float64), np_of(back)[1][:, None].astype(np.float64)
    assert np.linalg.norm(keys[:, 0] - ref.stored(turned[:, heads], fmt)) <= 1e-3 * np.linalg.norm(keys)  # a quant may be another
    for rows, out_type, total in ((3, torch.float32, None), (150, torch.bfloat16, 1024)):
        q = (rng.standard_normal((total or rows, heads, hd)) * 2).astype(np.float32)
        qd, out = torch_of(q.reshape(len(q), -1)), torch.zeros(len(q), heads * hd, device="cuda", dtype=out_type)
        b, hold = batch(rows, total)
        cache.attend(b, heads, qd.data_ptr(), 0, heads * hd, out.data_ptr(), int(out_type == torch.bfloat16), heads * hd, hd ** -0.5,
                     window, work.data_ptr())
        assert capi.kernel_status(0) == 0
        want = ref.attention(q[:rows], keys, vals, appended, hd ** -0.5, window)
        bound = ref.fp32_norm_bound(2.0) if total is None else ref.norm_bound(hd, 2.0, 1.0, True)
        got = np_of(out)[:rows].reshape(rows, heads, hd)
        assert np.linalg.norm(got - want) <= np.linalg.norm(want) * bound


# ---- what cannot be right is reported -------------------------------------------------------------------------------------

def status_of(call):
    call()
    with pytest.raises(capi.QmmError) as e:
        capi.kernel_status(0)
    assert e.value.code == capi.E_KERNEL and capi.kernel_status(0) == 0
    return str(e.value)


@pytest.mark.parametrize("fmt", FMTS)
def test_bad_pages_and_rows_are_skipped_and_reported(fmt):
    import torch
    rng = np.random.default_rng(16)
    p = Paged(fmt, 1, 64, 16, [40, 40])
    ks, vs = p.fill(rng)
    pool = p.pool.clone()
    good = p.table_dev.clone()
    x = torch_of(rng.standard_normal((4, 64)).astype(np.float32))
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    qd, out = torch_of(q.reshape(2, -1)), torch.zeros(2, 128, device="cuda")

    def append(b):
        p.cache.append(b, None, 0, 0, 0, 0, x.data_ptr(), 64, x.data_ptr(), 64, 0, 0, 0)

    def attend(b):
        p.cache.attend(b, 2, qd.data_ptr(), 0, 128, out.data_ptr(), 0, 128, 0.125, 0, p.workspace.data_ptr())

    for page in (-1, p.n_pages, 2 ** 31 - 1):
        p.table_dev[0, 2] = page
        assert "21" in status_of(lambda: append(p.batch([2, 0], [40, 40])))
        assert "21" in status_of(lambda: attend(p.batch([1, 1], [40, 40], single=True)))
        want = ref.attention(q[1:], ks[1], vs[1], 40, 0.125)  # the other sequence is as ever
        assert np.abs(np_of(out)[1].reshape(2, 64) - want[0]).max() <= ref.attention_bound(q, ks[1], vs[1], 0.125, False)
    p.table_dev.copy_(good)
    for rows, lens, begin in (([1, 1], [49, 40], None), ([1, 1], [-1, 40], None), ([1, 1], [40, 40], [0, -5, 2]),
                              ([1, 1], [40, 40], [0, 9, 2])):
        b = p.batch(rows, lens)
        if begin is not None:
            t = torch.tensor(begin, dtype=torch.int32, device="cuda")
            p.hold.append(t)
            b.row_begin_dev = t.data_ptr()
        assert "22" in status_of(lambda: attend(b))
    assert "22" in status_of(lambda: append(p.batch([4], [3])))  # rows in front of the first token
    assert torch.equal(p.pool, pool)
    assert int(p.workspace[:16384].to(torch.int32).sum()) == 0
    got = p.attend(q, [1, 1], [40, 40], 2, single=True)          # and the next call is whole
    for s in range(2):
        want = ref.attention(q[s:s + 1], ks[s], vs[s], 40, 0.125)
        assert np.abs(got[s] - want[0]).max() <= ref.attention_bound(q, ks[s], vs[s], 0.125, False)


@pytest.mark.parametrize("fmt", FMTS)
def test_bad_pages_and_rows_among_many_rows(fmt):
    """Whole tiles at a time: what is bad is left out and reported, the rest is stored."""
    import torch
    rng = np.random.default_rng(26)
    rows, hd = [420, 0, 420], 64
    p = Paged(fmt, 1, hd, 32, [440, 3, 420])
    x = torch_of(rng.standard_normal((840, hd)).astype(np.float32))
    back = torch.full((2, 840, hd), 5.0, device="cuda")

    def append(b):
        p.cache.append(b, None, 0, 0, 0, 0, x.data_ptr(), hd, x.data_ptr(), hd, 0, 0, 0)

    def read(b):
        p.cache.read(b, back[0].data_ptr(), hd, back[1].data_ptr(), hd, 0)

    b = p.batch(rows, p.lens)
    good = int(p.table_dev[0, 4])
    for page in (-1, p.n_pages, 2 ** 31 - 1):
        p.table_dev[0, 4] = page  # positions 128 to 159, rows 108 to 139
        assert "21" in status_of(lambda: append(b))
        assert "21" in status_of(lambda: read(b))
    want = ref.stored(x.cpu().numpy().reshape(840, 1, hd), fmt).astype(np.float32)[:, 0]
    want[108:140] = 5.0
    np.testing.assert_array_equal(np_of(back)[0], want)
    np.testing.assert_array_equal(np_of(back)[1], want)
    p.table_dev[0, 4] = good
    pool = p.pool.clone()
    for lens, begin in (([419, 3, 419], None), ([-1, 3, 2 ** 30], None), ([440, 3, 420], [0, -3, 2 ** 30, 840]),
                        ([440, 3, 420], [9, 4, 2, -1])):
        b = p.batch(rows, lens)
        if begin is not None:
            t = torch.tensor(begin, dtype=torch.int32, device="cuda")
            p.hold.append(t)
            b.row_begin_dev = t.data_ptr()
        assert "22" in status_of(lambda: append(b))
        assert "22" in status_of(lambda: read(b))
    assert torch.equal(p.pool, pool)


@pytest.mark.parametrize("n", [8, 900])
def test_sequences_that_cannot_be_right_are_reported_without_rows_of_their_own(n):
    import torch
    hd = 64
    p = Paged(ref.Q8_0, 1, hd, 16, [n, n, n])
    x = torch_of(np.ones((n, hd), np.float32))
    back = torch.zeros(2, n, hd, device="cuda")
    for begin, lens in (([0, 4, 2, 2], [n] * 3), ([0, 4, n + 1, n + 1], [n] * 3), ([0, 4, 4, -1], [n] * 3), ([-1, -1, 0, n], [n] * 3),
                        ([0, n, n, n], [n, -1, n]), ([0, n, n, n], [n, n, p.width * 16 + 1])):
        b = p.batch([n], lens)
        t = torch.tensor(begin, dtype=torch.int32, device="cuda")
        b.row_begin_dev = t.data_ptr()
        assert "22" in status_of(lambda: p.cache.append(b, None, 0, 0, 0, 0, x.data_ptr(), hd, x.data_ptr(), hd, 0, 0, 0))
        assert "22" in status_of(lambda: p.cache.read(b, back[0].data_ptr(), hd, back[1].data_ptr(), hd, 0))


def test_empty_calls_do_nothing():
    p = Paged(ref.Q4_0, 1, 64, 16, [4])
    b = capi.KVBatch(0, p.width, p.table_dev.data_ptr(), p.table_dev.data_ptr(), 0, 0)
    p.cache.append(b, None, 0, 0, 0, 0, 0, 64, 0, 64, 0, 0, 0)
    p.cache.read(b, 0, 64, 0, 64, 0)
    p.cache.attend(b, 2, 0, 0, 128, 0, 0, 128, 0.125, 0, 0)
    assert capi.kernel_status(0) == 0 and math.isfinite(1.0)
