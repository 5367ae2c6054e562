"""The 8-bit paged cache on the GPU: kv8_append bit by bit and kv8_attention within its bound against kv8_reference.py."""
import numpy as np
import pytest
import torch

import kv8_reference as ref
from glm_asr_stack_b200 import engine, ops

pytestmark = pytest.mark.gpu


class Batch:
    """A pool with random pages, and sequences with `new[i]` new tokens behind `ctx[i]` cached ones."""

    def __init__(self, new, ctx, kv_heads=2, group=4, page=16, seed=0, spread=1.0, fill=True, missing=()):
        self.rng = np.random.default_rng(seed)
        self.new, self.ctx, self.lens = list(new), list(ctx), [a + b for a, b in zip(new, ctx)]
        self.kv_heads, self.heads, self.page, self.group = kv_heads, kv_heads * group, page, group
        need = [-(-max(n, 0) // page) for n in self.lens]
        self.blocks = sum(need) + 2
        perm = self.rng.permutation(self.blocks).tolist()
        self.tables = np.full((len(new), max(need + [1]) + 1), -1, dtype=np.int32)
        for i, n in enumerate(need):
            self.tables[i, :n] = [perm.pop() for _ in range(n)]
        for i, j in missing:
            self.tables[i, j] = -1
        shape = (self.blocks, kv_heads, page, ref.DIM)
        self.codes, self.scales = [], []
        for _ in range(2):
            c = self.rng.integers(0, 256, shape).astype(np.uint8)
            c[(c & 127) == 127] ^= 1                          # no NaN codes
            e = self.rng.integers(-3, 4, shape[:2] + (page // ref.GROUP,)) if fill else np.zeros(shape[:2] + (page // ref.GROUP,))
            self.codes.append(c)
            self.scales.append((spread * 2.0 ** (e - 7.0)).astype(np.float32))
        self.total = sum(self.new)
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)

    def rows(self, heads, spread=1.0, extra=0):
        return ref.bf16(self.rng.normal(size=(self.total + extra, heads, ref.DIM)) * spread)

    def device(self):
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        k, v = (up(c).view(torch.float8_e4m3fn) for c in self.codes)
        ks, vs = (up(s) for s in self.scales)
        return (k, v, ks, vs), up(self.tables), torch.tensor(self.lens, dtype=torch.int32, device="cuda"), up(self.cu)


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda().to(torch.bfloat16)


def same_bits(a, b):
    return np.array_equal(a.view(np.uint32 if a.dtype == np.float32 else np.uint8), b.view(np.uint32 if b.dtype == np.float32 else np.uint8))


def check_append(b, key, value, theta, query=None, qout=None, pool=None):
    """Compare the pool after an append with the reference's, and the queries with their rotation."""
    want_c, want_s = [c.copy() for c in b.codes], [s.copy() for s in b.scales]
    for i, n in enumerate(b.new):
        rows = slice(int(b.cu[i]), int(b.cu[i]) + n)
        if n:
            ref.append(want_c[0], want_s[0], key[rows], b.tables[i], b.lens[i] - n, theta, b.page)
            ref.append(want_c[1], want_s[1], value[rows], b.tables[i], b.lens[i] - n, None, b.page)
    k, v, ks, vs = (t.cpu() for t in pool)
    for got, want in ((ks, want_s[0]), (vs, want_s[1])):
        assert np.array_equal(np.isnan(got.numpy()), np.isnan(want)) and np.array_equal(np.nan_to_num(got.numpy()), np.nan_to_num(want))
    assert same_bits(v.view(torch.uint8).numpy(), want_c[1])
    # -0 and +0 are one value: cos and sin may differ in the last bit of 64, and so may the sign of what they cancel to
    got = k.view(torch.uint8).numpy()
    assert np.array_equal(np.where(got == 128, 0, got), np.where(want_c[0] == 128, 0, want_c[0]))
    if query is not None:
        for i, n in enumerate(b.new):
            for t in range(n):
                p = b.lens[i] - n + t
                if p < 0:
                    continue
                q = query[b.cu[i] + t]
                want = ref.rotate(q, p, theta)
                mag = np.abs(np.concatenate([q[:, :64]] * 2, 1)) + np.abs(np.concatenate([q[:, 64:]] * 2, 1))
                # half a bf16 step, and three fp32 roundings of at most the two products' size
                tol = 2.0 ** -8 * np.abs(want) + 3 * 2.0 ** -24 * mag * (1 + 2.0 ** -8) + 1e-38
                assert np.all(np.abs(qout[b.cu[i] + t].float().cpu().numpy() - want) <= tol)
    b.codes, b.scales = want_c, want_s


@pytest.mark.parametrize("new,ctx", [([1], [0]), ([1], [15]), ([1, 1, 1], [16, 31, 300]), ([16], [0]), ([17, 0, 5], [15, 40, 0]), ([50, 3], [7, 100_003]),
                                     ([0, 0, 33], [0, 9, 1])])
@pytest.mark.parametrize("kv_heads,group,page", [(4, 4, 16), (1, 3, 48), (2, 1, 64)])
def test_append(new, ctx, kv_heads, group, page):
    b = Batch(new, ctx, kv_heads, group, page)
    q, k, v = b.rows(b.heads), b.rows(kv_heads, 3.0), b.rows(kv_heads)
    pool, tables, lens, cu = b.device()
    qo = ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu, query=dev(q))
    check_append(b, k, v, 10000.0, q, qo, pool)


def test_append_slices_of_a_projection_in_place_without_rotation_and_without_queries():
    b = Batch([5, 30], [3, 0], 2, 4, 16)
    qkv = b.rows(b.heads + 4)
    q, k, v = qkv[:, :b.heads], qkv[:, b.heads:b.heads + 2], qkv[:, b.heads + 2:]
    pool, tables, lens, cu = b.device()
    d = dev(np.concatenate([qkv, qkv], axis=1))               # a wider pitch than the rows need
    h = b.heads
    got = ops.kv8_append(*pool, d[:, h:h + 2], d[:, h + 2:h + 4], tables, lens, cu, query=d[:, :h], query_out=d[:, :h], theta=500.0)
    check_append(b, k, v, 500.0, q, got, pool)
    assert torch.equal(d[:, h:].cpu().float(), torch.from_numpy(np.concatenate([qkv, qkv], axis=1)[:, h:]).float())
    # theta 0: as they come; the same tokens again leave everything as it is
    b2 = Batch([20], [9], 2, 4, 16, seed=3)
    k, v = b2.rows(2), b2.rows(2)
    pool, tables, lens, cu = b2.device()
    assert ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu, theta=0.0) is None
    check_append(b2, k, v, 0, pool=pool)
    before = [t.clone() for t in pool]
    ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu, theta=0.0)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, pool))


def test_append_token_by_token_as_scales_grow():
    b = Batch([1, 1], [0, 5], 1, 1, 16, seed=1)
    sizes = [0.0, 1e-39, 3e-30, 1e-3, 1e-3, 7.0, 3.0, 900.0, 1e5, 1e19, 4e20, 2.0, 1.0, 1.0, 1.0, 1.0, 5.0, 0.0]
    for step, size in enumerate(sizes):
        k, v = b.rows(1) * size, b.rows(1) * size
        k, v = ref.bf16(k), ref.bf16(v)
        pool, tables, lens, cu = b.device()
        ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu)
        check_append(b, k, v, 10000.0, pool=pool)
        b.lens = [n + 1 for n in b.lens]
        if max(b.lens) > b.tables.shape[1] * 16 or b.tables[0, (b.lens[0] - 1) // 16] < 0 or b.tables[1, (b.lens[1] - 1) // 16] < 0:
            free = [x for x in range(b.blocks) if x not in b.tables]
            for i in range(2):
                j = (b.lens[i] - 1) // 16
                if b.tables[i, j] < 0:
                    b.tables[i, j] = free.pop()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan, 3e38])
def test_append_a_value_that_is_not_finite_poisons_its_block_until_it_starts_anew(bad):
    b = Batch([4, 4], [5, 14], 2, 2, 16, seed=2)
    k, v = b.rows(2), b.rows(2)
    k[1, 1, 70], v[5, 0, 3] = bad, bad                        # sequence 0 head 1; sequence 1 head 0, position 15
    pool, tables, lens, cu = b.device()
    with np.errstate(invalid="ignore"):
        ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu)
        check_append(b, k, v, 10000.0, pool=pool)
    assert np.isnan(b.scales[0]).sum() == 1 and np.isnan(b.scales[1]).sum() == 1
    b.lens, b.new = [10, 4], [1, 4]                           # one more behind the poisoned block; from the start
    b.cu, b.total = np.array([0, 1, 5], dtype=np.int32), 5
    k, v = b.rows(2), b.rows(2)
    pool, tables, lens, cu = b.device()
    ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu)
    check_append(b, k, v, 10000.0, pool=pool)
    assert np.isnan(b.scales[0]).sum() == 1


def test_append_leaves_alone_what_is_not_its_own():
    b = Batch([3, 2, 4], [14, 2, 20], 2, 4, 16, missing=[(0, 1), (2, 1)])
    q, k, v = (b.rows(n, extra=3) for n in (b.heads, 2, 2))
    pool, tables, lens, cu = b.device()
    tables[1, 0] = b.blocks + 5                               # no such page
    b.tables[1, 0] = -1
    lens[2] = 2                                               # two of its four new tokens are before position 0
    b.lens[2] = 2
    qo = torch.full((b.total + 3, b.heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu, query=dev(q), query_out=qo)
    check_append(b, k, v, 10000.0, q, qo, pool)
    assert torch.all(qo[b.total:] == 7) and torch.all(qo[5:7] == 7)


def attend(b, q, window=0, sinks=0, **more):
    pool, tables, lens, cu = b.device()
    out = torch.full((q.shape[0], q.shape[1], 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv8_attention(dev(q), *pool, tables, lens, cu, window=window, sinks=sinks, out=out, **more)
    assert ops.status() == 0
    return out


def check_attention(b, q, out, window=0, sinks=0, rows=None, **more):
    for i, n in enumerate(b.new):
        if not n:
            continue
        r = slice(int(b.cu[i]), int(b.cu[i]) + n)
        take = range(n) if rows is None else [t for t in rows if t < n]
        for t in take:
            want, tol = ref.attend(q[r][t:t + 1], b.codes[0], b.scales[0], b.codes[1], b.scales[1], b.tables[i], b.lens[i] - n + t + 1, window, sinks, **more)
            got = out[r][t:t + 1].float().cpu().numpy()
            bad = np.abs(got - want) > tol
            assert not bad.any(), (i, t, np.argwhere(bad)[0], got[bad][0], want[bad][0], tol[bad][0])


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 257, 300, 511, 513]


@pytest.mark.parametrize("kv_heads,group,page", [(4, 4, 16), (2, 1, 48), (1, 8, 64), (1, 16, 16), (1, 20, 32), (2, 3, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 3), (16, 16), (100, 40), (5000, 4)])
def test_one_query_each(kv_heads, group, page, window, sinks):
    b = Batch([1] * len(LENGTHS), [n - 1 for n in LENGTHS], kv_heads, group, page)
    q = b.rows(b.heads)
    # the longest length to expect chooses how the work is dealt out, and nothing else
    for max_len in (513, 40_000):
        check_attention(b, q, attend(b, q, window, sinks, max_new=1, max_len=max_len), window, sinks)


@pytest.mark.parametrize("new,ctx", [([5, 0, 3, 1], [40, 70, 0, 299]), ([8, 7], [120, 500]), ([2], [1000]), ([9, 9, 9], [0, 15, 16])])
@pytest.mark.parametrize("kv_heads,group", [(4, 4), (1, 2), (1, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 2)])
def test_a_few_queries_each(new, ctx, kv_heads, group, window, sinks):
    b = Batch(new, ctx, kv_heads, group, 16)
    q = b.rows(b.heads, extra=2)
    # max_new below what comes: several tiles of rows; right; far above: the kernel for many queries
    for max_new, max_len in ((1, 2000), (max(new), 600), (max(new), 50_000), (100_000, 600)):
        out = attend(b, q, window, sinks, max_new=max_new, max_len=max_len)
        check_attention(b, q, out, window, sinks)
        assert torch.all(out[b.total:] == 7)


@pytest.mark.parametrize("new,ctx", [([33], [0]), ([129, 40], [0, 250]), ([70, 1, 0, 300], [511, 600, 8, 0])])
@pytest.mark.parametrize("kv_heads,group,page", [(2, 4, 16), (1, 1, 64), (1, 20, 32), (1, 3, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 5), (200, 33)])
def test_many_queries_each(new, ctx, kv_heads, group, page, window, sinks):
    b = Batch(new, ctx, kv_heads, group, page)
    q = b.rows(b.heads, extra=1)
    for more in ({}, {"max_new": 100_000}):
        out = attend(b, q, window, sinks, **more)
        check_attention(b, q, out, window, sinks, rows=[0, 1, 2, 31, 32, 33, 41, 69, 127, 128, 131, 171, 299])
        assert torch.all(out[b.total:] == 7)


def test_short_and_long_sequences_together():
    """Contexts of a tile or less between long ones, cut into pieces that begin and end anywhere."""
    rng = np.random.default_rng(8)
    ctx = [int(n) for n in np.where(rng.random(60) < 0.8, rng.integers(0, 140, 60), rng.integers(2000, 5000, 60))]
    for new, group in ((1, 4), (1, 8), (4, 8)):
        b = Batch([new] * 60, ctx, 2, group, 16, missing=[(5, 0)])
        b.lens[7] = b.lens[40] = 0                            # nothing to see
        q = b.rows(b.heads)
        check_attention(b, q, attend(b, q, max_new=new, max_len=5000))


@pytest.mark.parametrize("kv_heads,group", [(4, 4), (4, 8), (2, 16)])
def test_more_contexts_than_places_for_them(kv_heads, group):
    """CTAs take over further contexts, the longest first: each is worked on once, whatever the lengths and the hints."""
    rng = np.random.default_rng(9)
    n = 330
    new = (rng.random(n) < 0.9).astype(int).tolist()
    b = Batch(new, rng.integers(0, 420, n).tolist(), kv_heads, group, 16)
    b.lens[3] = b.lens[200] = 0
    q = b.rows(b.heads)
    seen = torch.tensor([n == 1 and m > 0 for n, m in zip(new, b.lens)])[torch.tensor(new) == 1]
    for max_len in (1, 500):
        out = attend(b, q, max_new=1, max_len=max_len)
        assert torch.equal(torch.any(out != 0, dim=2).all(1).cpu(), seen)
        for i in range(3, n, 17):
            for r in range(int(b.cu[i]), int(b.cu[i + 1])):
                want, tol = ref.attend(q[r:r + 1], b.codes[0], b.scales[0], b.codes[1], b.scales[1], b.tables[i], b.lens[i])
                assert np.all(np.abs(out[r:r + 1].float().cpu().numpy() - want) <= tol)
    more = Batch([3] * 150, rng.integers(0, 2500, 150).tolist(), kv_heads, group, 16)      # longer, and more rows, than said
    q = more.rows(more.heads)
    out = attend(more, q, max_new=1, max_len=100)
    for i in range(0, 150, 19):
        for t in range(3):
            r = slice(3 * i + t, 3 * i + t + 1)
            want, tol = ref.attend(q[r], more.codes[0], more.scales[0], more.codes[1], more.scales[1], more.tables[i], more.lens[i] - 2 + t)
            assert np.all(np.abs(out[r].float().cpu().numpy() - want) <= tol)
    assert not torch.any(torch.all(out[:more.total] == 0, dim=2))


def test_rows_of_a_projection_and_into_wider_rows():
    b = Batch([3, 0, 70], [20, 4, 9], 2, 4, 16)
    q = b.rows(b.heads + 4)
    pool, tables, lens, cu = b.device()
    for max_new in (3, 100_000):
        out = torch.full((b.total + 2, 2 * b.heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        got = ops.kv8_attention(dev(q)[:, 2:2 + b.heads], *pool, tables, lens, cu, max_new=max_new, out=out[:b.total, b.heads:])
        check_attention(b, q[:, 2:2 + b.heads], got, rows=[0, 1, 2, 33, 69])
        assert torch.all(out[:, :b.heads] == 7) and torch.all(out[b.total:] == 7)


def test_a_prefix_that_sequences_share():
    b = Batch([1, 2, 1], [200, 150, 90], 2, 4, 16)
    b.tables[1, :6], b.tables[2, :5] = b.tables[0, :6], b.tables[0, :5]
    q = b.rows(b.heads)
    for max_new, max_len in ((2, 300), (2, 50_000), (100_000, 300)):
        check_attention(b, q, attend(b, q, max_new=max_new, max_len=max_len))


@pytest.mark.parametrize("new,ctx", [(1, 40), (2, 7)])
def test_more_sequences_than_one_line_of_work_has(new, ctx):
    n = 4500
    b = Batch([new] * n, [ctx + i % 30 for i in range(n)], 1, 2, 16)
    q, k, v = b.rows(2), b.rows(1), b.rows(1)
    out = attend(b, q, max_new=new, max_len=80)
    pool, tables, lens, cu = b.device()
    for i in range(0, n, 113):
        r = slice(int(b.cu[i]), int(b.cu[i]) + new)
        for t in range(new):
            want, tol = ref.attend(q[r][t:t + 1], b.codes[0], b.scales[0], b.codes[1], b.scales[1], b.tables[i], b.lens[i] - new + t + 1)
            assert np.all(np.abs(out[r][t:t + 1].float().cpu().numpy() - want) <= tol)
    ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu)
    check_append(b, k, v, 10000.0, pool=pool)


def test_a_pool_of_more_than_4_gib():
    """Pages whose byte offset in the pool does not fit 32 bits."""
    b = Batch([1, 20, 90], [70, 33, 5], 1, 4, 16)
    first = (1 << 32) // (16 * 128) + 7
    small, tables, lens, cu = b.device()
    big = tuple(torch.empty((first + b.blocks,) + t.shape[1:], dtype=t.dtype, device="cuda") for t in small)
    for x, t in zip(big, small):
        x[first:].view(torch.uint8).copy_(t.view(torch.uint8))
    tables = torch.where(tables >= 0, tables + first, tables)
    q, k, v = b.rows(4), b.rows(1), b.rows(1)
    for max_new in (1, 100_000):
        out = ops.kv8_attention(dev(q), *big, tables, lens, cu, max_new=max_new)
        check_attention(b, q, out, rows=[0, 1, 19, 77, 89])
    ops.kv8_append(*big, dev(k), dev(v), tables, lens, cu)
    check_append(b, k, v, 10000.0, pool=tuple(t[first:] for t in big))
    assert ops.status() == 0


def test_a_batch_without_a_new_token():
    """All of the packed rows lie behind the last sequence: nothing is read, written or appended."""
    b = Batch([0, 0, 0], [5, 0, 40], 2, 4, 16)
    pool, tables, lens, cu = b.device()
    before = [t.clone() for t in pool]
    q, kv = (torch.full((9, h, 128), float("nan"), dtype=torch.bfloat16, device="cuda") for h in (8, 2))
    for max_new, max_len in ((1, 100), (1, 50_000), (100_000, 100)):
        out = torch.full_like(q, 7.0)
        ops.kv8_attention(q, *pool, tables, lens, cu, max_new=max_new, max_len=max_len, out=out)
        assert torch.all(out == 7)
    qo = torch.full_like(q, 7.0)
    ops.kv8_append(*pool, kv, kv, tables, lens, cu, query=q, query_out=qo)
    assert torch.all(qo == 7) and all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, pool))
    assert ops.status() == 0


@pytest.mark.parametrize("new", [1, 7, 90])
def test_pages_a_window_has_left_behind(new):
    b = Batch([new, new], [400, 333], 2, 4, 16)
    for i in range(2):
        for j in range(2, (b.ctx[i] - 60 + 1) // 16):         # no query sees them; the first two have the first tokens
            b.tables[i, j] = -1 if j % 2 else b.blocks + 9
    q = b.rows(b.heads)
    full = Batch([new, new], [400, 333], 2, 4, 16)
    for max_new, max_len in ((new, 500), (new, 50_000), (100_000, 500)):
        out = attend(b, q, 60, 20, max_new=max_new, max_len=max_len)
        check_attention(full, q, out, 60, 20, rows=[0, 1, 6, 31, 60, 89])


@pytest.mark.parametrize("new", [1, 3, 70])
def test_what_is_not_there(new):
    """Missing pages, lengths below the number of new tokens, positions behind the table: not seen, and what lies in unused
    places of the pool -- NaN codes and NaN scales -- does not matter."""
    b = Batch([new] * 4, [100, 37, 60, 9], 2, 4, 16, missing=[(0, 0), (0, 3), (2, 1)])
    b.tables[3, :] = -1                                       # no page at all: zeros
    b.lens[1] = new - 1 if new > 1 else 0                     # the first query is before position 0
    used = np.zeros((b.blocks, 16), dtype=bool)
    for i in range(4):
        for p in range(b.lens[i]):
            if b.tables[i, p // 16] >= 0:
                used[b.tables[i, p // 16], p % 16] = True
    for c, s in zip(b.codes, b.scales):
        c[np.broadcast_to(~used[:, None, :, None], c.shape)] = 0x7F
        s[np.broadcast_to(~used.any(1)[:, None, None], s.shape)] = np.nan
    q = b.rows(b.heads)
    for max_new in (new, 200):
        out = attend(b, q, max_new=max_new, max_len=200)
        check_attention(b, q, out)
        assert torch.all(out[3 * new:] == 0)
    # a length the table has no pages for
    b2 = Batch([2], [30], 1, 4, 16)
    pool, tables, lens, cu = b2.device()
    q = b2.rows(4)
    out = ops.kv8_attention(dev(q), *pool, tables[:, :1].contiguous(), lens, cu)
    b2.tables = b2.tables[:, :1]
    check_attention(b2, q, out)


@pytest.mark.parametrize("new", [1, 4, 100])
def test_a_poisoned_block_reaches_those_who_see_it_only(new):
    b = Batch([new, new], [140, 140], 2, 2, 16)
    first = 140 // 16 - 2                                     # a block that a window of 30 has left behind for the last queries
    b.scales[0][b.tables[0, first], 1], b.codes[0][b.tables[0, first], 1] = np.nan, 0
    last = (140 + new - 1) // 16                              # the last block: only queries in it see it
    b.scales[1][b.tables[1, last], 0], b.codes[1][b.tables[1, last], 0] = np.nan, 0
    q = b.rows(b.heads)
    for window in (0, 30):
        out = attend(b, q, window, 0, max_new=new, max_len=300).float().cpu().numpy()
        for i in range(2):
            for t in range(new):
                p = 140 + t
                lo = max(0, p - window + 1) if window else 0
                want = np.zeros(4, dtype=bool)
                if i == 0:
                    want[2:] = lo <= first * 16 + 15
                else:
                    want[:2] = p >= last * 16
                got = np.isnan(out[i * new + t])
                assert np.array_equal(got.all(1), want) and np.array_equal(got.any(1), want), (window, i, t)


@pytest.mark.parametrize("new", [1, 4, 60])
@pytest.mark.parametrize("span", [8, 30, 60])
def test_scales_far_apart(new, span):
    """Blocks whose V, and K, are up to 2^span times the others': weights and sums keep their precision."""
    b = Batch([new, new], [200, 77], 1, 4, 16, seed=span)
    b.scales[1] *= (2.0 ** b.rng.integers(-span, 1, b.scales[1].shape)).astype(np.float32)
    b.scales[0] *= (2.0 ** b.rng.integers(-6, 3, b.scales[0].shape)).astype(np.float32)
    q = b.rows(4)
    q[0] *= 2.0 ** -100
    q[-1] = 0
    check_attention(b, q, attend(b, q, max_new=new, max_len=300), rows=[0, 1, 3, 17, 40, 59])


def test_scale_argument_and_queries_that_are_not_finite():
    b = Batch([1, 1, 1, 1], [100, 100, 100, 100], 1, 4, 16)
    q = b.rows(4)
    q[1, 2, 5], q[2, 0, 0] = np.inf, np.nan
    pool, tables, lens, cu = b.device()
    for max_new in (1, 200):
        out = ops.kv8_attention(dev(q), *pool, tables, lens, cu, max_new=max_new, scale=0.02)
        bad = torch.isnan(out.float()).all(dim=2).cpu().numpy()
        want = np.zeros((4, 4), dtype=bool)
        want[1, 2] = want[2, 0] = True
        assert np.array_equal(bad, want)
        keep = [0, 3]
        for i in keep:
            w, tol = ref.attend(q[i:i + 1], b.codes[0], b.scales[0], b.codes[1], b.scales[1], b.tables[i], b.lens[i], scale=float(np.float32(0.02)))
            assert np.all(np.abs(out[i:i + 1].float().cpu().numpy() - w) <= tol)


def test_a_prompt_then_steps_and_drafts():
    """The calls as a program makes them: a prompt in two pieces, steps of one token, a step with drafts of which some are taken
    back, through a pool of two layers; every call against the cache that the reference keeps."""
    layers, kv_heads, group, page = 2, 2, 4, 16
    rng = np.random.default_rng(5)
    pool = engine.KV8Pool(24, page, layers, kv_heads)
    tables = rng.permutation(24)[:22].reshape(2, 11).astype(np.int32)
    d_tables = torch.from_numpy(tables).cuda()
    caches = [[[np.zeros((24, kv_heads, page, 128), dtype=np.uint8), np.zeros((24, kv_heads, 1), dtype=np.float32)] for _ in range(2)] for _ in range(layers)]
    have = [0, 0]
    for new, keep in (([37, 21], None), ([40, 1], None), ([1, 1], None), ([1, 1], None), ([5, 4], [2, 3]), ([1, 1], None)):
        lens = [a + b for a, b in zip(have, new)]
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        d_lens, d_cu = torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.from_numpy(cu).cuda()
        for layer in range(layers):
            qkv = ref.bf16(rng.normal(size=(sum(new), (group + 2) * kv_heads, 128)))
            d = dev(qkv)
            h = group * kv_heads
            q = ops.kv8_append(*pool.layer(layer), d[:, h:h + kv_heads], d[:, h + kv_heads:], d_tables, d_lens, d_cu, query=d[:, :h])
            out = ops.kv8_attention(q, *pool.layer(layer), d_tables, d_lens, d_cu, max_new=max(new), max_len=max(lens))
            (kc, ks), (vc, vs) = caches[layer]
            for i in range(2):
                r = slice(int(cu[i]), int(cu[i + 1]))
                ref.append(kc, ks, qkv[r, h:h + kv_heads], tables[i], have[i], 10000.0, page)
                ref.append(vc, vs, qkv[r, h + kv_heads:], tables[i], have[i], None, page)
                for t in range(new[i]):
                    want, tol = ref.attend(q[cu[i] + t:cu[i] + t + 1].double().cpu().numpy(), kc, ks, vc, vs, tables[i], have[i] + t + 1)
                    assert np.all(np.abs(out[cu[i] + t:cu[i] + t + 1].float().cpu().numpy() - want) <= tol)
        have = [a + (b if keep is None else keep[i]) for i, (a, b) in enumerate(zip(have, new))]
    assert ops.status() == 0


@pytest.mark.parametrize("new,max_len", [(1, 300), (1, 50_000), (6, 50_000), (80, 300)])
def test_captured_replayed_and_on_another_stream(new, max_len):
    """Two graphs of the same calls, replayed with other lengths, at once on two streams: as the eager calls."""
    b = Batch([new] * 3, [200, 17, 90], 2, 4, 16)
    q, k, v = dev(b.rows(b.heads)), dev(b.rows(2)), dev(b.rows(2))
    graphs = []
    for g in range(2):
        pool, tables, lens, cu = b.device()
        out = torch.zeros_like(q)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        ops.set_stream(s)
        try:
            with torch.cuda.stream(s):
                def run():
                    r = ops.kv8_append(*pool, k, v, tables, lens, cu, query=q)
                    ops.kv8_attention(r, *pool, tables, lens, cu, max_new=new, max_len=max_len, out=out)
                run()
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=s):
                    run()
        finally:
            ops.set_stream(None)
        graphs.append((graph, s, pool, lens, out, tables, cu))
    for shift in (0, 3, -9):
        fresh = b.device()
        for (graph, s, pool, lens, out, _, _), d in zip(graphs, (shift, shift + 1)):
            for t, f in zip(pool, fresh[0]):
                t.copy_(f)
            lens.copy_(fresh[2] + d)
        torch.cuda.synchronize()
        for graph, s, *_ in graphs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (graph, s, pool, lens, out, tables, cu), d in zip(graphs, (shift, shift + 1)):
            eager, _, l2, _ = b.device()
            l2 = l2 + d
            r = ops.kv8_append(*eager, k, v, tables, l2, cu, query=q)
            want = ops.kv8_attention(r, *eager, tables, l2, cu, max_new=new, max_len=max_len)
            assert torch.equal(out, want)
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(pool, eager))
    assert ops.status() == 0


def test_repeatable():
    b = Batch([1] * 40, list(range(1, 2000, 50)), 4, 4, 16)
    q = b.rows(b.heads)
    for more in ({"max_new": 1, "max_len": 300}, {"max_new": 1, "max_len": 50_000}, {"max_new": 100}):
        first = attend(b, q, **more)
        assert all(torch.equal(first, attend(b, q, **more)) for _ in range(3))


def test_refusals():
    b = Batch([2, 1], [5, 6], 2, 4, 16)
    pool, tables, lens, cu = b.device()
    k, v, ks, vs = pool
    q, key = dev(b.rows(8)), dev(b.rows(2))
    run = lambda *a, **m: ops.kv8_append(*a, **m)  # noqa: E731
    att = lambda *a, **m: ops.kv8_attention(*a, **m)  # noqa: E731
    bad = [
        (TypeError, lambda: run(*pool, key.float(), key, tables, lens, cu)),
        (TypeError, lambda: run(k.float(), v, ks, vs, key, key, tables, lens, cu)),
        (TypeError, lambda: run(k, v, ks.double(), vs, key, key, tables, lens, cu)),
        (TypeError, lambda: run(*pool, key, key, tables.long(), lens, cu)),
        (TypeError, lambda: att(q.half(), *pool, tables, lens, cu)),
        (ValueError, lambda: run(*pool, key, key[:2], tables, lens, cu)),
        (ValueError, lambda: run(*pool, key, key, tables, lens, cu, query=q[:2])),
        (ValueError, lambda: run(*pool, key, key, tables, lens, cu, query_out=q)),
        (ValueError, lambda: run(*pool, q, q, tables, lens, cu)),
        (ValueError, lambda: run(*pool, key, key, tables, lens, cu[:2])),
        (ValueError, lambda: run(*pool, key, key, tables[:1], lens, cu)),
        (ValueError, lambda: run(*pool, key, key, tables, lens, cu, theta=-1.0)),
        (ValueError, lambda: run(k, v[:1], ks, vs, key, key, tables, lens, cu)),
        (ValueError, lambda: run(k, v, ks[:1], vs, key, key, tables, lens, cu)),
        (ValueError, lambda: run(*pool, key.transpose(0, 1), key.transpose(0, 1), tables, lens, cu)),
        (ValueError, lambda: run(*pool, key.cpu(), key, tables, lens, cu)),
        (ValueError, lambda: run(*pool, key, key, tables, lens.cpu(), cu)),
        (ValueError, lambda: att(q[:, :7], *pool, tables, lens, cu)),
        (ValueError, lambda: att(q[:, :, :64], *pool, tables, lens, cu)),
        (ValueError, lambda: att(q, *pool, tables, lens, cu, out=q)),
        (ValueError, lambda: att(q, *pool, tables, lens, cu, out=q[:2].clone())),
        (ValueError, lambda: att(q, *pool, tables, lens, cu, window=-1)),
        (ValueError, lambda: att(q, *pool, tables, lens, cu, sinks=-1)),
        (ValueError, lambda: att(q, *pool, tables, lens, cu, scale=float("inf"))),
        (ValueError, lambda: att(q, *pool, tables, lens, cu, scale=-0.1)),
        (ValueError, lambda: att(q, *pool, tables, lens, cu, max_new=-1)),
    ]
    before = [t.clone() for t in pool]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, pool))
    # nothing to do
    none = torch.zeros((0, 8, 128), dtype=torch.bfloat16, device="cuda")
    assert att(none, *pool, tables, lens, torch.zeros_like(cu)).shape == (0, 8, 128)
    assert run(*pool, none[:, :2], none[:, :2], tables, lens, torch.zeros_like(cu)) is None
    assert ops.status() == 0
