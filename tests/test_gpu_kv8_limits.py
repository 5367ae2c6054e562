"""The 8-bit paged cache where its numbers, streams and forms of work reach their limits, against kv8_reference.py."""
import numpy as np
import pytest
import torch

import kv8_reference as ref
from glm_asr_stack_b200 import _lib, ops
from test_gpu_kv8 import Batch, check_append, check_attention, dev

pytestmark = pytest.mark.gpu

LN2 = float(np.float32(np.log(2.0)))
STRETCH = 1 + 2.0 ** -5


def ladder(steps, tokens, new, seed=0):
    """One sequence whose i-th run of 64 keys has the score STRETCH * steps[i][0] (log2, under the scale ln 2: no power of two, which
    any format holds) and the V scale steps[i][1]; the score and scale of the last run last to the end."""
    b = Batch([new], [tokens - new], 1, 4, 16, seed=seed)
    k, v, ks, vs = b.codes[0], b.codes[1], b.scales[0], b.scales[1]
    k[...], ks[...] = 0, 1.0
    for g in range(-(-tokens // 16)):
        score, scale = steps[min(g // 4, len(steps) - 1)]
        blk = b.tables[0, g]
        k[blk, 0, :, 0] = ref.e4m3(np.array([float(score)]))[0]
        assert ref.VALUE[k[blk, 0, 0, 0]] == score
        vs[blk] = scale
        if scale in (0.0, 2.0 ** -126):
            v[blk] = 0
    q = np.zeros((new, b.heads, ref.DIM))
    q[:, :, 0] = STRETCH
    return b, q


def bound(b, q, row):
    """The result, and how far a kernel may be from it: weights off by 2^-8 of themselves (twice, above and below the line), scores
    exact here but for 2^-20, the bf16 result by half a step.  Small weights may be off by 2^-20 of the largest PRODUCT of weight
    and V scale, or by 2^-25 of the largest weight under the V scales within 2^5 of the smallest that a key here has: neither
    lets a small weight on a large value go."""
    want, _ = ref.attend(q[row:row + 1], b.codes[0], b.scales[0], b.codes[1], b.scales[1], b.tables[0], b.lens[0] - b.new[0] + row + 1, scale=LN2)
    length = b.lens[0] - b.new[0] + row + 1
    at = np.arange(length)
    blk = b.tables[0, at // 16]
    x = STRETCH * ref.VALUE[b.codes[0][blk, 0, at % 16, 0]]
    w = np.exp((x - x.max()) * LN2)
    w /= w.sum()
    vs = b.scales[1][blk, 0, 0].astype(np.float64)
    codes = np.abs(ref.VALUE[b.codes[1][blk, 0, at % 16]])
    small = 2.0 ** -20 * (w * vs).max() + 2.0 ** -25 * w.max() * min(vs.max(), vs.min() * 2.0 ** 5)
    return want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -19) * 2 * ((w * vs) @ codes)[None, None] + small * codes.sum(0)[None, None] + 1e-37


LADDERS = {
    "up 2^16": [(16, 1.0), (0, 2.0 ** 16)],
    "up 2^20": [(20, 1.0), (0, 2.0 ** 20)],
    "up 2^24": [(24, 1.0), (0, 2.0 ** 24)],
    "up 2^30": [(30, 1.0), (0, 2.0 ** 30)],
    "down 2^24": [(0, 2.0 ** 24), (24, 1.0)],
    "up 2^4 eleven times": [(4 * (11 - i), 2.0 ** (4 * i)) for i in range(12)],
    "up 2^2 fourteen times": [(2 * (14 - i), 2.0 ** (2 * i)) for i in range(15)],
    "up, down and up": [(24, 1.0), (0, 2.0 ** 24), (24, 1.0), (0, 2.0 ** 24)],
    "zeros first": [(26, 2.0 ** -126), (0, 1.0)],
    "never written first": [(26, 0.0), (0, 1.0)],
    "zeros last": [(0, 1.0), (26, 2.0 ** -126)],
    "far out": [(30, 2.0 ** -60), (0, 2.0 ** -30), (-30, 1.0)],
}


@pytest.mark.parametrize("name", LADDERS)
@pytest.mark.parametrize("new", [1, 40])
def test_v_scales_that_change_along_the_context(name, new):
    """Small weights on large values, in every order, by both kernels: the hint chooses between them and not the result."""
    steps = LADDERS[name]
    tokens = 64 * len(steps) + 70 + new
    b, q = ladder(steps, tokens, new)
    pool, tables, lens, cu = b.device()
    for max_new in (1, 100_000):
        out = ops.kv8_attention(dev(q), *pool, tables, lens, cu, max_new=max_new, scale=LN2).float().cpu().numpy()
        for row in {0, new // 2, new - 1}:
            want, tol = bound(b, q, row)
            assert np.all(np.abs(out[row:row + 1] - want) <= tol), (max_new, row, (np.abs(out[row:row + 1] - want) / tol).max())
    assert ops.status() == 0


def test_slices_that_overlap_are_refused():
    b = Batch([3, 2], [20, 4], 2, 4, 16)
    pool, tables, lens, cu = b.device()
    buf = dev(b.rows(3 * b.heads, extra=1))
    h, n = b.heads, b.total
    before = [buf.clone()] + [t.clone() for t in pool]
    for out in (buf[:n, 1:1 + h], buf[1:, :h], buf[1:, h - 1:2 * h - 1], buf[:n, :h]):
        with pytest.raises(ValueError):
            ops.kv8_attention(buf[:n, :h], *pool, tables, lens, cu, out=out)
    kv = buf[:n, 2 * h:2 * h + 2]
    for query, out, key, value in ((0, 1, kv, kv), (0, h, buf[:n, h:h + 2], kv), (0, h, kv, buf[:n, 2 * h - 2:2 * h]), (0, h, kv, buf[1:, h + 1:h + 3])):
        with pytest.raises(ValueError):
            ops.kv8_append(*pool, key, value, tables, lens, cu, query=buf[:n, query:query + h], query_out=buf[:n, out:out + h])
    torch.cuda.synchronize()
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, [buf, *pool]))
    # side by side in one array
    apart = ops.kv8_attention(buf[:n, :h].clone(), *pool, tables, lens, cu)
    assert torch.equal(ops.kv8_attention(buf[:n, :h], *pool, tables, lens, cu, out=buf[:n, h:2 * h]), apart)
    assert torch.equal(buf[:, :h], before[0][:, :h]) and torch.equal(buf[:, 2 * h:], before[0][:, 2 * h:])


@pytest.mark.parametrize("own_stream", [False, True])
def test_what_a_call_allocates_belongs_to_the_stream_that_works_on_it(own_stream):
    """torch's current stream is another one than the launches'.  Blocks that the current stream's pool has back are still in use on it,
    and a result that is dropped at once is still being written: no call may touch the one or give the other away."""
    b = Batch([1] * 3, [5000, 17, 90], 2, 4, 16)
    pool, tables, lens, cu = b.device()
    q, k = dev(b.rows(b.heads)), dev(b.rows(2))
    want_q = ops.kv8_append(*pool, k, k, tables, lens, cu, query=q)
    want = ops.kv8_attention(want_q, *pool, tables, lens, cu, max_new=1)
    size = _lib.load().glmasr_kv8_attention_workspace()
    other = torch.cuda.Stream()
    current, launch = (torch.cuda.default_stream(), other) if own_stream else (other, torch.cuda.default_stream())
    rest = lambda s: s.synchronize() or torch.cuda._sleep(40_000_000)  # noqa: E731  about 20 ms
    torch.cuda.synchronize()
    if own_stream:
        ops.set_stream(other)
    try:
        with torch.cuda.stream(current):
            for nbytes in (size, q.numel() * 2):
                used = torch.full((nbytes,), 7, dtype=torch.uint8, device="cuda")
                rest(current)
                copy = used.clone()                           # when the current stream gets to it
                del used
                q2 = ops.kv8_append(*pool, k, k, tables, lens, cu, query=q)
                got = ops.kv8_attention(want_q, *pool, tables, lens, cu, max_new=1)
                torch.cuda.synchronize()
                assert torch.all(copy == 7)
                assert torch.equal(got, want) and torch.equal(q2, want_q)
                del copy, q2, got
            for call in (lambda: ops.kv8_append(*pool, k, k, tables, lens, cu, query=q), lambda: ops.kv8_attention(want_q, *pool, tables, lens, cu, max_new=1)):
                with torch.cuda.stream(launch):
                    rest(launch)
                call()                                        # its result is dropped while the launch stream is still asleep
                after = torch.full_like(q, 5.0)
                torch.cuda.synchronize()
                assert torch.all(after == 5)
                del after
    finally:
        ops.set_stream(None)
    assert ops.status() == 0


@pytest.mark.parametrize("new,ctx", [([1], [0]), ([1, 5], [7, 300]), ([40, 2], [3, 15])])
def test_no_rotation_leaves_every_bit_of_the_queries(new, ctx):
    """theta = 0: a dim has nothing from its partner, be that infinite or no number, and a zero keeps its sign."""
    b = Batch(new, ctx, 2, 4, 16)
    q, k = dev(b.rows(b.heads)), dev(b.rows(2))
    flat = q.view(b.total, -1)
    for i, x in enumerate((np.inf, -np.inf, np.nan, -0.0, 3e38)):
        flat[:, 7 + 65 * i] = x
    q = flat.view(q.shape)
    pool, tables, lens, cu = b.device()
    want = q.clone()
    got = ops.kv8_append(*pool, k, k, tables, lens, cu, query=q, theta=0.0)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    wide = torch.cat([q, q], dim=1)                           # in place, into rows of a wider pitch
    ops.kv8_append(*pool, k, k, tables, lens, cu, query=wide[:, :b.heads], query_out=wide[:, :b.heads], theta=0.0)
    assert torch.equal(wide.view(torch.int16), torch.cat([want, want], dim=1).view(torch.int16))


# Keys below 2^-126 whose rotation lies within 2^-150 of the middle between two codes: position, dim, and the two elements in
# units of 2^-133
NEXT_TO_A_BORDER = [(2783, 28, 101, -94), (344, 42, -79, -51), (220, 38, 46, 34), (2835, 43, -49, 105), (1625, 38, -89, -114), (1199, 49, -36, 67),
                    (3258, 55, -71, -78), (1235, 62, 46, 45), (1550, 53, 58, 54), (3907, 7, -39, -90), (4773, 63, -39, -115), (1646, 23, -35, -78)]


def test_keys_below_the_smallest_normal_number_next_to_a_border():
    n = len(NEXT_TO_A_BORDER)
    b = Batch([1] * n, [p for p, *_ in NEXT_TO_A_BORDER], 1, 2, 16)
    for i, (p, *_) in enumerate(NEXT_TO_A_BORDER):            # earlier tokens of the block: scale 2^-126 as well
        b.scales[0][b.tables[i, p // 16]] = 2.0 ** -126
    k = np.zeros((n, 1, ref.DIM))
    for i, (_, d, x, y) in enumerate(NEXT_TO_A_BORDER):
        k[i, 0, d], k[i, 0, d + 64] = x * 2.0 ** -133, y * 2.0 ** -133
    v = b.rows(1)
    pool, tables, lens, cu = b.device()
    ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu)
    check_append(b, k, v, 10000.0, pool=pool)


def test_numbers_that_do_not_fit_32_bits():
    """A window, first tokens and expectations beyond every length there is: no limit, as 2^31 - 1 is, and not their low 32 bits."""
    b = Batch([2, 1], [100, 50], 2, 4, 16)
    q = b.rows(b.heads)
    pool, tables, lens, cu = b.device()
    want = ops.kv8_attention(dev(q), *pool, tables, lens, cu)
    check_attention(b, q, want)
    for far in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 16, 2 ** 40 + 3):
        assert torch.equal(ops.kv8_attention(dev(q), *pool, tables, lens, cu, window=far), want), far
        assert torch.equal(ops.kv8_attention(dev(q), *pool, tables, lens, cu, window=5, sinks=far), want), far
        out = ops.kv8_attention(dev(q), *pool, tables, lens, cu, max_new=far, max_len=far)
        check_attention(b, q, out)
    for bad in ({"window": -2 ** 32 + 5}, {"window": 5, "sinks": -2 ** 32}, {"max_new": -2 ** 32 + 1}, {"max_len": -2 ** 32 + 1}):
        with pytest.raises(ValueError):
            ops.kv8_attention(dev(q), *pool, tables, lens, cu, **bad)


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 16, 2 ** 31 - 17, -1, -2 ** 31, -2 ** 31 + 1])
def test_a_length_that_cannot_be_is_its_own_sequence_s_concern(length):
    """Behind every table, or below zero: nothing of it is written, and the sequences around it are as without it."""
    b = Batch([2, 1, 3, 1], [40, 50, 20, 7], 2, 4, 16)
    q, k, v = b.rows(b.heads), b.rows(2), b.rows(2)
    pool, tables, lens, cu = b.device()
    lens[1] = length
    qo = torch.full((b.total, b.heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv8_append(*pool, dev(k), dev(v), tables, lens, cu, query=dev(q), query_out=qo)
    around = [0, 1, 3, 4, 5, 6]
    got = qo[around]
    b.new[1], b.tables[1] = 0, -1                             # the same batch without it
    keep = np.array(around)
    b.cu, b.total = np.array([0, 2, 2, 5, 6], dtype=np.int32), 6
    check_append(b, k[keep], v[keep], 10000.0, q[keep], got, pool)
    for max_new in (1, 100_000):
        out = ops.kv8_attention(qo, *pool, tables, lens, cu, max_new=max_new)
        check_attention(b, got.double().cpu().numpy(), out[around])
        assert length > 0 or not torch.any(out[2])
    assert ops.status() == 0


def in_pieces(b, q, columns, **more):
    """The attention of a batch whose table has room for so many pages that a context is cut into pieces, which a second launch joins."""
    pool, tables, lens, cu = b.device()
    tables = torch.nn.functional.pad(tables, (0, max(0, columns - tables.shape[1])), value=-1)
    out = torch.full((q.shape[0], b.heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    before = ops.launch_count()
    ops.kv8_attention(dev(q), *pool, tables, lens, cu, max_len=50_000, out=out, **more)
    assert ops.launch_count() - before == 2
    assert ops.status() == 0
    return out


LENGTHS = [1, 2, 15, 16, 17, 33, 127, 128, 129, 300, 513, 2049, 2500]


@pytest.mark.parametrize("kv_heads,group,page", [(4, 4, 16), (2, 1, 48), (1, 8, 64), (1, 20, 32), (2, 3, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2100, 0), (2100, 40), (2200, 2300), (5000, 4)])
def test_pieces_of_contexts(kv_heads, group, page, window, sinks):
    """One query each; a window of more than 16 tiles, so that pieces begin and end before, in and behind what it leaves out."""
    b = Batch([1] * len(LENGTHS), [n - 1 for n in LENGTHS], kv_heads, group, page)
    q = b.rows(b.heads)
    check_attention(b, q, in_pieces(b, q, 5120 // page, max_new=1, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("new", [1, 2, 4, 7])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2100, 100), (2100, 1)])
def test_pieces_with_a_gap_between_the_first_tokens_and_the_window(new, window, sinks):
    b = Batch([new] * 3, [4100, 3333, 2101], 1, 4, 16)
    q = b.rows(b.heads, extra=2)
    out = in_pieces(b, q, 320, max_new=new, window=window, sinks=sinks)
    check_attention(b, q, out, window, sinks)
    assert torch.all(out[b.total:] == 7)


def test_pieces_of_few_units_over_all_blocks():
    """Fewer groups than blocks, more sequences than blocks, and sequences without any."""
    for ctx in ([700], [3000, 0], [17] * 500, [0] * 30 + [2600] + [0] * 30):
        b = Batch([1] * len(ctx), ctx, 2, 4, 16)
        q = b.rows(b.heads)
        check_attention(b, q, in_pieces(b, q, 400, max_new=1))


def test_pieces_of_a_batch_without_a_new_token():
    b = Batch([0, 0, 0], [5, 0, 40], 2, 4, 16)
    out = in_pieces(b, np.full((9, 8, 128), np.nan), 400, max_new=1)
    assert torch.all(out == 7)


@pytest.mark.parametrize("new", [1, 3])
def test_pieces_of_a_prefix_that_sequences_share(new):
    b = Batch([new, 2, 1], [2000, 1500, 900], 2, 4, 16)
    b.tables[1, :60], b.tables[2, :50] = b.tables[0, :60], b.tables[0, :50]
    q = b.rows(b.heads)
    check_attention(b, q, in_pieces(b, q, 400, max_new=new))


@pytest.mark.parametrize("new", [1, 3, 7])
def test_pieces_with_pages_that_are_not_there(new):
    """Missing pages from the first to the last, a whole piece of them, none at all; lengths below the new tokens; and what lies in places
    that nothing is in does not matter."""
    b = Batch([new] * 5, [2500, 700, 1900, 9, 40], 2, 4, 16, missing=[(0, 0), (0, 3), (2, 1), (2, 110), (1, 20)] + [(0, j) for j in range(30, 90)])
    b.tables[3, :] = -1
    b.tables[2, 60:70] = b.blocks + 5
    b.lens[4] = new - 1
    used = np.zeros((b.blocks, 16), dtype=bool)
    for i in range(5):
        for p in range(b.lens[i]):
            if 0 <= b.tables[i, p // 16] < b.blocks:
                used[b.tables[i, p // 16], p % 16] = True
    for c, s in zip(b.codes, b.scales):
        c[np.broadcast_to(~used[:, None, :, None], c.shape)] = 0x7F
        s[np.broadcast_to(~used.any(1)[:, None, None], s.shape)] = np.nan
    q = b.rows(b.heads)
    out = in_pieces(b, q, 400, max_new=new)
    check_attention(b, q, out)
    assert torch.all(out[3 * new:4 * new] == 0)


@pytest.mark.parametrize("new", [1, 4])
def test_pieces_of_pages_a_window_has_left_behind(new):
    b = Batch([new, new], [4000, 3333], 2, 4, 16)
    for i in range(2):
        for j in range(2, (b.ctx[i] - 2200 + 1) // 16):
            b.tables[i, j] = -1 if j % 2 else b.blocks + 9
    q = b.rows(b.heads)
    full = Batch([new, new], [4000, 3333], 2, 4, 16)
    check_attention(full, q, in_pieces(b, q, 400, max_new=new, window=2200, sinks=20), 2200, 20)


@pytest.mark.parametrize("new", [1, 4])
@pytest.mark.parametrize("which", [0, 1])
def test_pieces_with_a_poisoned_block(new, which):
    """In the first, a middle and the last piece of a context: every query that sees it, and no other."""
    for place in (0, 60, (2000 + new - 1) // 16):
        b = Batch([new, new], [2000, 2000], 2, 2, 16)
        b.scales[which][b.tables[0, place], 1], b.codes[which][b.tables[0, place], 1] = np.nan, 0
        q = b.rows(b.heads)
        got = torch.isnan(in_pieces(b, q, 400, max_new=new)).cpu().numpy()
        want = np.zeros((2 * new, 4), dtype=bool)
        for t in range(new):
            want[t, 2:] = 2000 + t >= place * 16
        assert np.array_equal(got.all(2), want) and np.array_equal(got.any(2), want)
        # a window that has left it behind
        if place == 60:
            assert not torch.any(torch.isnan(in_pieces(b, q, 400, max_new=new, window=1000)))


@pytest.mark.parametrize("new", [1, 4])
@pytest.mark.parametrize("span", [8, 30, 60])
def test_pieces_of_scales_far_apart(new, span):
    """The parts of a context have references far from each other."""
    b = Batch([new, new], [2000, 1077], 1, 4, 16, seed=span)
    run = np.repeat(b.rng.integers(-span, 1, -(-b.blocks // 7)), 7)[:b.blocks]
    for i in range(2):                                        # some 110 tokens in a row under one scale
        n = (b.tables[i] >= 0).sum()
        b.scales[1][b.tables[i, :n]] = (2.0 ** run[:n].astype(np.float64))[:, None, None]
    b.scales[0] *= (2.0 ** b.rng.integers(-6, 3, b.scales[0].shape)).astype(np.float32)
    q = b.rows(4)
    q[0] *= 2.0 ** -100
    q[-1] = 0
    check_attention(b, q, in_pieces(b, q, 400, max_new=new))


@pytest.mark.parametrize("name", LADDERS)
def test_pieces_of_v_scales_that_change_along_the_context(name):
    """As whole contexts have them: a part's small weights on large values count in the whole."""
    steps = LADDERS[name]
    b, q = ladder(steps, 64 * len(steps) + 70 + 3, 3)
    out = in_pieces(b, q, 400, max_new=3, scale=LN2).float().cpu().numpy()
    for row in range(3):
        want, tol = bound(b, q, row)
        assert np.all(np.abs(out[row:row + 1] - want) <= tol), (row, (np.abs(out[row:row + 1] - want) / tol).max())


@pytest.mark.parametrize("new", [1, 6])
def test_pieces_captured_replayed_and_on_two_streams(new):
    """Two graphs of an append and an attention in pieces, each with a workspace of its own, replayed at once on two streams with other
    lengths than they were captured with: as the eager calls."""
    b = Batch([new] * 3, [2000, 17, 900], 2, 4, 16)
    q, k, v = dev(b.rows(b.heads)), dev(b.rows(2)), dev(b.rows(2))
    wide = lambda t: torch.nn.functional.pad(t, (0, 400 - t.shape[1]), value=-1)  # noqa: E731
    graphs = []
    for g in range(2):
        pool, tables, lens, cu = b.device()
        tables = wide(tables)
        out = torch.zeros_like(q)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        ops.set_stream(s)
        try:
            with torch.cuda.stream(s):
                def run():
                    r = ops.kv8_append(*pool, k, v, tables, lens, cu, query=q)
                    ops.kv8_attention(r, *pool, tables, lens, cu, max_new=new, max_len=50_000, out=out)
                before = ops.launch_count()
                run()
                assert ops.launch_count() - before == 3
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=s):
                    run()
        finally:
            ops.set_stream(None)
        graphs.append((graph, s, pool, lens, out, tables, cu))
    for shift in (0, 3, -9, -900):
        fresh = b.device()
        for (graph, s, pool, lens, out, _, _), d in zip(graphs, (shift, shift + 1)):
            for t, f in zip(pool, fresh[0]):
                t.copy_(f)
            lens.copy_(torch.clamp(fresh[2] + d, min=new))
        torch.cuda.synchronize()
        for _ in range(3):                                    # the same tokens again leave the cache as it is
            for graph, s, *_ in graphs:
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, s, pool, lens, out, tables, cu in graphs:
            eager = b.device()[0]
            r = ops.kv8_append(*eager, k, v, tables, lens, cu, query=q)
            want = ops.kv8_attention(r, *eager, tables, lens, cu, max_new=new, max_len=50_000)
            assert torch.equal(out, want)
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(pool, eager))
    assert ops.status() == 0


def beside_a_sink(tokens, new, score, page=64, seed=0):
    """The first token has a score so far above the others' that it has nearly all the weight, and V codes of 0 in a block of ordinary ones:
    the result is what the others, one small weight each, add up to."""
    b = Batch([new], [tokens - new], 1, 4, page, seed=seed)
    k, v, ks, vs = b.codes[0], b.codes[1], b.scales[0], b.scales[1]
    k[...], ks[...], vs[...] = 0, 1.0, 1.0
    v[...] = ref.e4m3(b.rng.uniform(2.0, 3.5, v.shape))
    first = b.tables[0, 0]
    k[first, 0, 0, 0], v[first, 0, 0] = ref.e4m3(np.array([float(score)]))[0], 0
    assert ref.VALUE[k[first, 0, 0, 0]] == score
    q = np.zeros((new, b.heads, ref.DIM))
    q[:, :, 0] = STRETCH
    return b, q


def sink_bound(b, q, row, score):
    """Weights off by 2^-8 of themselves; small ones by half the step that they are held in, 2^-34 of the largest (f16 steps of 2^-24 below a
    reference of at least 2^9; e5m2 steps of 2^-16 over 2^6 below one of at least 2^12: 2^-35)."""
    length = b.lens[0] - b.new[0] + row + 1
    at = np.arange(length)
    v = ref.VALUE[b.codes[1][b.tables[0, at // b.page], 0, at % b.page]]
    w = np.full(length, 2.0 ** -(STRETCH * score))
    w[0] = 1.0
    w /= w.sum()
    want = w @ v
    return want, 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -19) * 2 * (w @ np.abs(v)) + 2.0 ** -34 * np.abs(v).sum(0)


@pytest.mark.parametrize("tokens,score", [(130, 14), (300, 18), (300, 22), (5000, 16), (5000, 20), (5000, 24), (30_000, 20), (30_000, 24), (30_000, 28)])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_many_small_weights_beside_one_that_has_nearly_all(tokens, score, new):
    b, q = beside_a_sink(tokens, new, score)
    pool, tables, lens, cu = b.device()
    for max_new in (1, 100_000):
        out = ops.kv8_attention(dev(q), *pool, tables, lens, cu, max_new=max_new, scale=LN2).float().cpu().numpy()
        for row in {0, new // 2, new - 1}:
            want, tol = sink_bound(b, q, row, score)
            assert np.all(np.abs(out[row] - want) <= tol), (max_new, row, (np.abs(out[row] - want) / tol).max(), (out[row] / want).mean())
    assert ops.status() == 0


@pytest.mark.parametrize("tokens,score", [(300, 22), (5000, 24)])
def test_pieces_with_many_small_weights_beside_one(tokens, score):
    b, q = beside_a_sink(tokens, 2, score)
    out = in_pieces(b, q, 400, max_new=2, scale=LN2).float().cpu().numpy()
    for row in range(2):
        want, tol = sink_bound(b, q, row, score)
        assert np.all(np.abs(out[row] - want) <= tol), (row, (np.abs(out[row] - want) / tol).max())
