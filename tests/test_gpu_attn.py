"""Attention operators over the paged int8 cache and packed prompts, against
their definitions in 64 bits (tests/attn_ref.py): types, head layouts, page
sizes, strides, empty and one-token sequences, masked NaN, bad indexes, side
streams, graphs, and a run of the three together."""
import numpy as np
import pytest
import torch

from attn_ref import (Cache, append, append_args, append_ref, check, decode, decode_ref, i32, prompt,
                      prompt_ref, rope_table, starts, status, within, workspace)

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def same_bits(a, b):
    """Equal as numbers, NaN where the other has NaN."""
    a, b = np.asarray(a), np.asarray(b)
    assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f"), np.argwhere(a != b)[:5]


# ------------------------------------------------------------------------------------- append

def run_append(cache, q, k, v, lengths, position, table, rope, n_rot, pairs, heads, out=F32,
               copies=True):
    """One call against the definition: codes, scales and copies, all equal."""
    T, D = k.shape[0], cache.dim
    want, rq, rk, rv = append_ref(cache, q, k, v, lengths, position, table, rope, n_rot, pairs)
    outs = [torch.full((T, n * D), 7.0, dtype=out, device="cuda") for n in (heads, cache.kv, cache.kv)]
    if q is None:
        outs[0] = None
    if not copies:
        outs[1] = outs[2] = None
    rope_d = torch.from_numpy(rope).cuda() if n_rot else None
    append(cache, append_args(q, k, v, starts(lengths), i32(position), i32(table), rope_d, n_rot,
                              pairs, out, *outs, heads=heads))
    torch.cuda.synchronize()
    assert status() == 0
    for got, ref in zip((cache.k, cache.ks, cache.v, cache.vs), want):
        same_bits(got.cpu().numpy(), ref)
    used = sum(lengths)
    for got, ref in zip(outs, (rq, rk, rv)):
        if got is not None:
            ref = torch.from_numpy(ref.reshape(used, -1)).to(out)
            same_bits(got[:used].float().cpu().numpy(), ref.float().numpy())
            assert (got[used:].float() == 7).all()  # rows of no sequence


@pytest.mark.parametrize("page,dim,kv,group,n_rot,pairs,dtype,out", [
    (16, 64, 3, 3, 64, 1, F32, F32), (32, 64, 3, 3, 64, 1, F32, F16),
    (64, 128, 5, 4, 128, 0, F32, F16), (128, 128, 1, 8, 128, 0, BF16, BF16),
    (16, 128, 2, 1, 64, 0, F16, F32), (128, 64, 2, 2, 16, 0, BF16, F16),
    (64, 64, 1, 12, 56, 0, F16, BF16), (32, 128, 3, 1, 120, 1, F32, BF16),
    (64, 128, 2, 2, 0, 0, BF16, F32), (32, 64, 2, 2, 6, 0, F32, F32), (32, 64, 2, 2, 10, 1, F16, F16),
    (64, 128, 2, 1, 2, 0, F32, F32), (128, 128, 2, 2, 126, 0, F32, F32),
])
def test_append_prompts_and_steps(page, dim, kv, group, n_rot, pairs, dtype, out):
    """New prompts and continued sequences of every length around a page's ends, empty ones between
    them, then single tokens."""
    g = gen(page + dim + n_rot)
    lengths = [1, 0, page - 1, page, page + 1, 3 * page + 5, 0, 2]
    position = [page + 3, 5, 0, page, 1, page - 1, 0, 2 * page - 1]
    need = [-(-(a + b) // page) for a, b in zip(lengths, position)]
    order = torch.randperm(sum(need) + 2, generator=gen(1), device="cuda").tolist()
    table, most = [], max(need) + 3
    for m in need:
        table.append([order.pop() for _ in range(m)] + [10 ** 6] * (most - m))  # entries never read
    cache = Cache(sum(need) + 2, page, kv, dim, fill=99)
    cache.ks.uniform_(0.001, 0.05, generator=g)
    cache.vs.uniform_(0.001, 0.05, generator=g)
    heads = kv * group
    rope = rope_table(max(a + b for a, b in zip(lengths, position)) + 4, n_rot, factor=2.5)
    T = sum(lengths) + 3  # rows behind the last sequence
    x = randn(g, T, (heads + 2 * kv) * dim, dtype=dtype)
    q, k, v = x.split([heads * dim, kv * dim, kv * dim], 1)  # strided: one fused projection
    run_append(cache, q, k, v, lengths, position, table, rope, n_rot, pairs, heads, out)
    position = [a + b for a, b in zip(lengths, position)]
    for s in range(len(need)):  # one more token may begin a page
        if position[s] // page >= need[s]:
            table[s][need[s]] = order.pop() if order else table[s][0]
    keep = [s for s in range(len(need)) if position[s] < need[s] * page]
    x = randn(g, len(keep), 2 * kv * dim, dtype=dtype) * 3
    k, v = x.split([kv * dim, kv * dim], 1)
    run_append(cache, None, k, v, [1] * len(keep), [position[s] for s in keep], [table[s] for s in keep],
               rope, n_rot, pairs, heads, out, copies=False)


@pytest.mark.parametrize("dim,dtype", [(64, F32), (128, BF16), (128, F32)])
def test_append_one_prompt_among_many_steps(dim, dtype):
    """A call made for single tokens that brings one long prompt as well: its pages hold more rows than
    the threads that such a call gets keep in registers."""
    g = gen(4)
    page, kv, group, n_rot = 128, 3, 2, 64
    lengths = [1] * 60 + [150] + [1] * 130
    position = [int(x) for x in np.random.default_rng(1).integers(0, 2 * page, len(lengths))]
    need = [-(-(a + b) // page) for a, b in zip(lengths, position)]
    order = torch.randperm(sum(need), generator=gen(2), device="cuda").tolist()
    table = [[order.pop() for _ in range(m)] + [0] * (max(need) - m) for m in need]
    c = Cache(sum(need), page, kv, dim, fill=3)
    c.ks.uniform_(0.001, 0.05, generator=g)
    c.vs.uniform_(0.001, 0.05, generator=g)
    T = sum(lengths)
    q, k, v = (randn(g, T, n * dim, dtype=dtype) for n in (kv * group, kv, kv))
    run_append(c, q, k, v, lengths, position, table, rope_table(3 * page + 200, n_rot), n_rot, 0, kv * group, F16)


def test_append_token_by_token_stays_within_a_step():
    """A page filled one token at a time with ever larger values: every value within one step of the
    page's last scale, and within half a step where the page was written by one call."""
    g = gen(5)
    page, kv, dim = 64, 2, 64
    x = randn(g, page, 2 * kv * dim) * torch.linspace(0.1, 40, page, device="cuda")[:, None]
    x[:8] = 0  # a page whose scale is zero at first
    k, v = x.split([kv * dim] * 2, 1)
    rope = rope_table(page, 0)
    for whole in (True, False):
        c = Cache(1, page, kv, dim)
        for t in range(1 if whole else page):
            rows = slice(0, page) if whole else slice(t, t + 1)
            run_append(c, None, k[rows], v[rows], [page if whole else 1], [t], [[0]], rope, 0, 0, kv,
                       copies=False)
        for codes, scale, src in ((c.k, c.ks, k), (c.v, c.vs, v)):
            got = codes[0].double() * scale[0].double()[:, None, None]
            off = (got.transpose(0, 1).reshape(page, -1) - src.double()).abs().view(page, kv, dim)
            steps = off / scale[0].double()[None, :, None]
            assert steps.max() <= (0.5001 if whole else 1.0), steps.max()


def test_append_not_finite_values_reach_the_scale():
    g = gen(6)
    page, kv, dim = 32, 3, 64
    c = Cache(4, page, kv, dim)
    k, v = randn(g, 5, kv * dim), randn(g, 5, kv * dim)
    k[2, 5] = float("nan")
    k[3, dim + 1] = float("inf")
    v[0, 2 * dim] = float("-inf")
    rope = rope_table(64, 64)
    run_append(c, None, k, v, [5], [3], [[2, 1]], rope, 64, 0, kv, copies=False)
    assert torch.isnan(c.ks[2]).tolist() == [True, True, False]
    assert torch.isnan(c.vs[2]).tolist() == [False, False, True]
    run_append(c, None, k[:1], k[:1], [1], [8], [[2, 1]], rope, 64, 0, kv, copies=False)
    assert torch.isnan(c.ks[2]).tolist() == [True, True, False]  # until the page is begun anew
    run_append(c, None, k[:1], k[:1], [1], [0], [[2, 1]], rope, 64, 0, kv, copies=False)
    assert not torch.isnan(c.ks[2]).any()


def test_append_tiny_and_huge_values():
    g = gen(7)
    page, kv, dim = 16, 1, 64
    rope = rope_table(16, 0)
    c = Cache(1, page, kv, dim)
    for t, size in enumerate((1e-43, 1e-38, 1e-20, 1.0, 1e30, 3e38)):
        x = (torch.rand(1, dim, generator=g, device="cuda") * 2 - 1) * size
        run_append(c, None, x, -x, [1], [t], [[0]], rope, 0, 0, kv, copies=False)


def test_append_bad_indexes_are_left_out_and_reported():
    """A page id, position or extent outside its range: nothing of that sequence's pages is written,
    the others are, and bit 2 of the device status says so."""
    g = gen(8)
    page, kv, dim = 16, 2, 64
    rope = torch.from_numpy(rope_table(64, 64)).cuda()
    k, v = randn(g, 6, kv * dim), randn(g, 6, kv * dim)
    good = Cache(4, page, kv, dim, fill=55)
    args = dict(q=None, k=k, v=v, rope=rope, n_rot=64, pairs=0, out_type=F32, heads=kv)
    append(good, append_args(start=i32([0, 3, 6]), position=i32([0, 0]), table=i32([[1, 1], [2, 2]]), **args))
    torch.cuda.synchronize()
    assert status() == 0
    for start, position, table in [
            ([0, 3, 6], [0, 0], [[1, 1], [4, 4]]),    # page id = number of pages
            ([0, 3, 6], [0, 0], [[1, 1], [-1, -1]]),  # negative page id
            ([0, 3, 6], [0, 30], [[1, 1], [2, 2]]),   # past its page table
            ([0, 3, 6], [0, -1], [[1, 1], [2, 2]]),   # negative position
            ([0, 3, 7], [0, 0], [[1, 1], [2, 2]]),    # past the call's tokens
            ([0, 3, 2], [0, 0], [[1, 1], [2, 2]]),    # descending
            ([0, 3, 2 ** 31 - 1], [0, 2 ** 31 - 1], [[1, 1], [2, 2]])]:
        c = Cache(4, page, kv, dim, fill=55)
        append(c, append_args(start=i32(start), position=i32(position), table=i32(table), **args))
        torch.cuda.synchronize()
        assert status() == 4 and status() == 0
        assert torch.equal(c.k[1], good.k[1]) and torch.equal(c.vs[1], good.vs[1])
        for p in (0, 2, 3):
            assert (c.k[p] == 55).all() and (c.v[p] == 55).all() and (c.ks[p] == 0).all()
    # a rotation table that is too short
    c = Cache(4, page, kv, dim, fill=55)
    append(c, append_args(start=i32([0, 3, 6]), position=i32([0, 0]), table=i32([[1, 1], [2, 2]]), **args,
                          rope_len=2))
    torch.cuda.synchronize()
    assert status() == 4 and (c.k == 55).all()


# ------------------------------------------------------------------------------------- decode

def filled(g, n_pages, page, kv, dim):
    c = Cache(n_pages, page, kv, dim)
    c.k.random_(-127, 128, generator=g)
    c.v.random_(-127, 128, generator=g)
    c.ks.uniform_(0.002, 0.03, generator=g)
    c.vs.uniform_(0.002, 0.03, generator=g)
    return c


def tables(g, lengths, page, spare=3):
    """A cache's size and page tables: pages in random order, ids behind a length out of range."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    most = max(need) + 2
    return total, [[order.pop() for _ in range(m)] + [-7] * (most - m) for m in need]


@pytest.mark.parametrize("page,dim,kv,group,dtype,out", [
    (16, 64, 3, 3, F32, F32), (32, 64, 3, 3, BF16, F32), (64, 64, 2, 1, F16, F16), (128, 64, 1, 8, F32, BF16),
    (16, 128, 5, 4, F32, F32), (32, 128, 2, 7, F16, F16), (64, 128, 5, 4, BF16, BF16),
    (128, 128, 1, 12, F32, F32), (64, 128, 1, 20, F16, F32), (64, 64, 1, 9, F32, F32),
])
def test_decode(page, dim, kv, group, dtype, out):
    g = gen(page * dim + group)
    lengths = [1, 0, page - 1, page, page + 1, 15, 16, 17, 700, 0, 2 * page, 333, 64, 63, 65, 129]
    total, table = tables(g, lengths, page)
    c = filled(g, total, page, kv, dim)
    heads = kv * group
    q = randn(g, len(lengths), heads * dim, dtype=dtype)
    q[3] *= 30  # one key takes nearly all the weight
    q[4] *= 0
    t = i32(table)
    got = decode(c, q, i32(lengths), t, heads, dim ** -0.5, out_type=out)
    torch.cuda.synchronize()
    assert status() == 0
    ref, tol = decode_ref(c, q, lengths, t, heads, dim ** -0.5)
    within(got, ref, tol)
    assert (got[1] == 0).all() and (got[9] == 0).all()


@pytest.mark.parametrize("lengths,kv,group,dim,page", [
    ([5000], 1, 4, 128, 64), ([20001], 5, 4, 128, 64), ([9000, 3, 0, 12345], 3, 3, 64, 32),
    ([70000, 1], 2, 8, 128, 128), ([4096] * 40, 8, 2, 64, 16),
    ([1] * 300, 2, 2, 128, 16), ([130] * 700, 1, 1, 64, 64),
])
def test_decode_long_and_many(lengths, kv, group, dim, page):
    g = gen(len(lengths) + lengths[0])
    total, table = tables(g, lengths, page)
    c = filled(g, total, page, kv, dim)
    heads = kv * group
    q = randn(g, len(lengths), heads * dim)
    t, n, ws = i32(table), i32(lengths), workspace(len(lengths), heads, c)
    got = decode(c, q, n, t, heads, dim ** -0.5, ws=ws)
    ref, tol = decode_ref(c, q, lengths, t, heads, dim ** -0.5)
    within(got, ref, tol)
    again = decode(c, q, n, t, heads, dim ** -0.5, ws=ws)  # the workspace is ready for the next call
    assert torch.equal(got, again)  # and the order of the sums is the same


def test_decode_strides_and_rows_beyond_the_lengths():
    """q and out inside wider rows; codes behind a length and scales of pages behind it do not count;
    what lies between the output rows stays."""
    g = gen(11)
    page, kv, group, dim = 32, 2, 3, 64
    heads, lengths = kv * group, [40, 7, 64]
    total, table = tables(g, lengths, page)
    c = filled(g, total, page, kv, dim)
    wide = randn(g, 3, heads * dim + 16)
    q = wide[:, 8:8 + heads * dim]
    out = torch.full((3, heads * dim + 32), 3.0, device="cuda")
    t = i32(table)
    ref, tol = decode_ref(c, q, lengths, t, heads, 0.2)
    decode(c, q, i32(lengths), t, heads, 0.2, out=out[:, 16:16 + heads * dim])
    within(out[:, 16:16 + heads * dim], ref, tol)
    assert (out[:, :16] == 3).all() and (out[:, 16 + heads * dim:] == 3).all()
    for s, n in enumerate(lengths):
        if n % page:
            for x in (c.k, c.v):
                x[table[s][n // page], :, n % page:] = -128
    spare = sorted(set(range(total)) - {p for r, n in zip(table, lengths) for p in r[:-(-n // page)]})
    c.ks[spare] = float("nan")
    c.vs[spare] = float("nan")
    t[:, 2] = spare[0]
    t[1, 1] = spare[0]
    once = out.clone()
    decode(c, q, i32(lengths), t, heads, 0.2, out=out[:, 16:16 + heads * dim])
    assert torch.equal(once, out)


def test_decode_one_workspace_for_every_shape():
    """Calls of other head sizes, batches and groups one after another over one workspace."""
    g = gen(16)
    ws = workspace(1, 1, Cache(1, 16, 1, 128))
    for page, dim, kv, group, lengths in [(16, 64, 2, 3, [5000, 3]), (64, 128, 5, 4, [700] * 30), (32, 128, 1, 9, [20000]),
                                          (128, 64, 3, 3, [1]), (16, 128, 2, 2, [0, 0]), (64, 64, 1, 1, [333] * 5)]:
        total, table = tables(g, lengths, page)
        c = filled(g, total, page, kv, dim)
        q = randn(g, len(lengths), kv * group * dim)
        t = i32(table)
        ref, tol = decode_ref(c, q, lengths, t, kv * group, 0.1)
        within(decode(c, q, i32(lengths), t, kv * group, 0.1, ws=ws), ref, tol)
    assert (ws[:1024] == 0).all()  # the counters


def test_calls_on_two_streams_at_once():
    """Decode over two caches, each with its own workspace, and a prompt, all in flight together."""
    g = gen(17)
    work = []
    for page, dim, kv, group, lengths in [(64, 128, 5, 4, [9000, 500, 20000]), (32, 64, 3, 3, [4000] * 20)]:
        total, table = tables(g, lengths, page)
        c = filled(g, total, page, kv, dim)
        q = randn(g, len(lengths), kv * group * dim)
        t = i32(table)
        work.append((c, q, i32(lengths), t, kv * group, workspace(len(lengths), kv * group, c),
                     decode_ref(c, q, lengths, t, kv * group, 0.1)))
    lengths = [700, 900]
    q, k, v = (randn(g, sum(lengths), n * 64, dtype=F16) for n in (4, 2, 2))
    pref, ptol = prompt_ref(q, k, v, lengths, 4, 2, 64, 0.1)
    start = starts(lengths)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [[], [], []]
    for _ in range(5):
        for i, (c, x, n, t, heads, ws, _) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                outs[i].append(decode(c, x, n, t, heads, 0.1, ws=ws))
        with torch.cuda.stream(streams[2]):
            outs[2].append(prompt(q, k, v, start, 4, 2, 64, 0.1))
    torch.cuda.synchronize()
    for i, w in enumerate(work):
        for o in outs[i]:
            within(o, *w[6])
    for o in outs[2]:
        within(o, pref, ptol)


def test_decode_not_finite():
    """A page whose scale is NaN shows in the heads that read it and in no others; an infinite or NaN
    query in its own head."""
    g = gen(12)
    page, kv, group, dim = 32, 2, 2, 64
    heads, lengths = kv * group, [100, 90]
    total, table = tables(g, lengths, page)
    c = filled(g, total, page, kv, dim)
    q = randn(g, 2, heads * dim)
    t = i32(table)
    ref, tol = decode_ref(c, q, lengths, t, heads, 0.2)
    c.ks[table[0][1], 0] = float("nan")
    c.vs[table[1][2], 1] = float("nan")
    got = decode(c, q, i32(lengths), t, heads, 0.2).view(2, heads, dim)
    ref, tol = ref.view(2, heads, dim), tol.view(2, heads, dim)
    assert torch.isnan(got[0, :2]).all() and torch.isnan(got[1, 2:]).all()
    within(got[0, 2:], ref[0, 2:], tol[0, 2:])
    within(got[1, :2], ref[1, :2], tol[1, :2])
    c2 = filled(gen(12), total, page, kv, dim)
    q[0, 3] = float("nan")
    q[1, dim + 3] = float("inf")
    got = decode(c2, q, i32(lengths), t, heads, 0.2).view(2, heads, dim)
    assert torch.isnan(got[0, 0]).all() and torch.isnan(got[1, 1]).all()
    assert torch.isfinite(got[0, 1:]).all() and torch.isfinite(got[1, 0]).all()


def test_decode_zero_scale_pages_and_wide_ranges():
    """Pages of zeros (scale 0), scales from 1e-30 to 1e30 among one sequence's pages, queries from
    1e-20 to 1e20 in size."""
    g = gen(13)
    page, kv, group, dim = 16, 1, 2, 64
    lengths = [100, 100, 100]
    total, table = tables(g, lengths, page)
    c = filled(g, total, page, kv, dim)
    c.ks[table[0][2]] = 0
    c.vs[table[0][3]] = 0
    c.vs[[table[1][j] for j in range(4)], 0] = torch.tensor([1e-30, 1e-10, 1.0, 1e30], device="cuda")
    q = randn(g, 3, group * dim)
    q[1] *= 1e-20
    q[2] *= 1e20
    c.ks[table[2][:7]] *= 1e-20
    t = i32(table)
    ref, tol = decode_ref(c, q, lengths, t, group, 0.1)
    within(decode(c, q, i32(lengths), t, group, 0.1), ref, tol)


def test_decode_bad_indexes_are_left_out_and_reported():
    g = gen(14)
    page, kv, group, dim = 32, 1, 2, 64
    lengths = [90, 40]
    total, table = tables(g, lengths, page)
    c = filled(g, total, page, kv, dim)
    q = randn(g, 2, group * dim)
    t = i32(table)
    good = decode(c, q, i32(lengths), t, group, 0.2)
    assert status() == 0
    for bad in (total, -1, 2 ** 31 - 1, -2 ** 31):
        u = t.clone()
        u[0, 1] = bad
        got = decode(c, q, i32(lengths), u, group, 0.2)
        assert status() == 4 and status() == 0
        assert torch.equal(got[1], good[1]) and torch.isfinite(got).all()
        # the page's keys take no part
        d = Cache(total, page, kv, dim)
        d.k, d.v, d.ks, d.vs = c.k, c.v, c.ks, c.vs
        ref, tol = decode_ref(d, q[:1], [58], torch.stack([t[0, 0], t[0, 2]])[None], group, 0.2)
        within(got[:1], ref, tol)
    for n in (-1, t.shape[1] * page + 1, 2 ** 31 - 1):
        got = decode(c, q, i32([n, 40]), t, group, 0.2)
        assert status() == 4
        assert torch.equal(got[1], good[1]) and (got[0] == 0).all()


def test_decode_offsets_past_32_bits():
    """Pages far apart in a cache of more than 2^31 bytes."""
    page, kv, dim = 128, 8, 128
    n_pages = (1 << 31) // (page * kv * dim) + 40
    g = gen(15)
    c = object.__new__(Cache)
    c.page, c.kv, c.dim = page, kv, dim
    c.k = torch.empty(n_pages, kv, page, dim, dtype=torch.int8, device="cuda")
    c.v = torch.empty_like(c.k)
    c.ks = torch.zeros(n_pages, kv, device="cuda")
    c.vs = torch.zeros(n_pages, kv, device="cuda")
    ids = [n_pages - 1, 0, n_pages - 30, n_pages // 2]
    k, v = randn(g, 450, kv * dim), randn(g, 450, kv * dim)
    append(c, append_args(None, k, v, i32([0, 450]), i32([0]), i32([ids]), None, 0, 0, F32, heads=kv))
    q = randn(g, 1, kv * dim)
    t = i32([ids])
    got = decode(c, q, i32([450]), t, kv, 0.1)
    ref, tol = decode_ref(c, q, [450], t, kv, 0.1)
    within(got, ref, tol)
    full = torch.softmax(torch.einsum("hd,thd->ht", q.double().view(kv, dim), k.double().view(-1, kv, dim)) * 0.1, -1)
    plain = torch.einsum("ht,thd->hd", full, v.double().view(-1, kv, dim))
    assert (got.view(kv, dim) - plain).abs().max() < 0.1  # the right rows, up to quantisation


# ------------------------------------------------------------------------------------- prompt

PROMPTS = [
    [1], [2, 0, 1, 31], [32, 33, 64], [0, 65, 127, 0, 128], [129, 1, 255, 256, 257], [700, 3, 383, 384, 385],
    [1030], [0, 0, 500, 0], [511, 512, 513],
]


@pytest.mark.parametrize("lengths", PROMPTS)
@pytest.mark.parametrize("heads,kv,dim,dtype", [(9, 3, 64, F16), (8, 2, 128, BF16), (5, 5, 128, F16),
                                                (6, 1, 64, BF16)])
def test_prompt(lengths, heads, kv, dim, dtype):
    g = gen(sum(lengths) + heads)
    T = sum(lengths) + 5  # rows behind the last sequence
    q = randn(g, T, heads * dim, dtype=dtype)
    k, v = randn(g, T, kv * dim, dtype=dtype), randn(g, T, kv * dim, dtype=dtype)
    out = torch.full((T, heads * dim), 3.0, dtype=dtype, device="cuda")
    got = prompt(q, k, v, starts(lengths), heads, kv, dim, dim ** -0.5, out=out)
    torch.cuda.synchronize()
    assert status() == 0
    ref, tol = prompt_ref(q, k, v, lengths, heads, kv, dim, dim ** -0.5)
    within(got[:T - 5], ref, tol)
    assert (got[T - 5:] == 3).all()


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16)])
def test_prompt_many_short_ones(dim, dtype):
    g = gen(21)
    rng = np.random.default_rng(3)
    lengths = rng.integers(0, 40, 300).tolist()
    T, heads, kv = sum(lengths), 4, 2
    q = randn(g, T, heads * dim, dtype=dtype)
    k, v = randn(g, T, kv * dim, dtype=dtype), randn(g, T, kv * dim, dtype=dtype)
    ref, tol = prompt_ref(q, k, v, lengths, heads, kv, dim, 0.1)
    within(prompt(q, k, v, starts(lengths), heads, kv, dim, 0.1), ref, tol)


@pytest.mark.parametrize("dim,dtype,scale", [(64, F16, 0.125), (128, BF16, 0.09), (64, BF16, 0.0),
                                             (128, F16, -0.07), (128, BF16, 1.5)])
def test_prompt_strides_f32_output_and_scales(dim, dtype, scale):
    """One fused projection's rows, an f32 output inside wider rows; a zero, a negative and a large scale."""
    g = gen(22)
    heads, kv, lengths = 4, 2, [150, 40, 300]
    T = sum(lengths)
    x = randn(g, T, (heads + 2 * kv) * dim + 8, dtype=dtype)
    q, k, v, _ = x.split([heads * dim, kv * dim, kv * dim, 8], 1)
    out = torch.full((T, heads * dim + 8), 3.0, device="cuda")
    prompt(q, k, v, starts(lengths), heads, kv, dim, scale, out=out[:, 4:4 + heads * dim])
    ref, tol = prompt_ref(q, k, v, lengths, heads, kv, dim, scale)
    within(out[:, 4:4 + heads * dim], ref, tol)
    assert (out[:, :4] == 3).all() and (out[:, 4 + heads * dim:] == 3).all()


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
def test_prompt_rising_scores(dim, dtype):
    """Each key outweighs all before it, so the running maximum moves at every step."""
    g = gen(23)
    heads, kv, lengths = 2, 1, [600]
    q = torch.ones(600, heads * dim, device="cuda", dtype=dtype)
    k = (torch.linspace(-6, 6, 600, device="cuda")[:, None] * torch.ones(dim, device="cuda")).to(dtype)
    v = randn(g, 600, dim, dtype=dtype)
    for scale in (1.0, -1.0):
        ref, tol = prompt_ref(q, k, v, lengths, heads, kv, dim, scale)
        within(prompt(q, k, v, starts(lengths), heads, kv, dim, scale), ref, tol)


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prompt_masked_rows_have_no_effect(dim, dtype, bad):
    """NaN or infinity in a key's or value's row reaches the rows that may see it, and no others: not
    the rows before it, not the neighbouring sequences."""
    g = gen(24)
    heads, kv, lengths = 4, 2, [70, 200, 90]
    T, at = sum(lengths), 70 + 150
    q = randn(g, T, heads * dim, dtype=dtype)
    k, v = randn(g, T, kv * dim, dtype=dtype), randn(g, T, kv * dim, dtype=dtype)
    ref, tol = prompt_ref(q, k, v, lengths, heads, kv, dim, 0.1)
    sees = torch.zeros(T, dtype=torch.bool, device="cuda")
    sees[at:270] = True
    for which in range(2):
        kk, vv = k.clone(), v.clone()
        (kk, vv)[which][at, dim + 3] = bad  # the second KV head
        got = prompt(q, kk, vv, starts(lengths), heads, kv, dim, 0.1)
        within(got[~sees], ref[~sees], tol[~sees])
        first = slice(0, 2 * dim)
        within(got[sees][:, first], ref[sees][:, first], tol[sees][:, first])
        mine = got[sees].view(-1, heads, dim)[:, 2:]
        if which == 0:
            # z is +-inf or NaN at that key: a weight of NaN, or (z = -inf) none at all
            z = q[sees].double().view(-1, heads, dim)[:, 2:, 3] * bad
            gone = z != -torch.inf
            assert torch.isnan(mine[gone]).all()
            if (~gone).any():
                without = torch.cat([torch.arange(70, at), torch.arange(at + 1, 270)])
                r, a = prompt_ref(q[without], k[without], v[without], [199], heads, kv, dim, 0.1)
                r, a = (y.view(-1, heads, dim)[149:, 2:] for y in (r, a))
                keep = ~gone[1:]
                within(mine[1:][keep], r[1:][keep], a[1:][keep])
        else:
            assert not torch.isfinite(mine[..., 3]).any()
            others = [i for i in range(dim) if i != 3]
            r, a = (y[sees].view(-1, heads, dim)[:, 2:][..., others] for y in (ref, tol))
            within(mine[..., others], r, a)


def test_prompt_captured_and_replayed():
    """A captured call replayed with other values and other borders between the sequences."""
    g = gen(26)
    heads, kv, dim, T = 4, 2, 128, 600
    q, k, v = (torch.empty(T, n * dim, dtype=BF16, device="cuda") for n in (heads, kv, kv))
    start = i32([0, 100, 100, 600])
    out = torch.empty(T, heads * dim, dtype=BF16, device="cuda")
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        prompt(q, k, v, start, heads, kv, dim, 0.1, out=out)
    for lengths in ([100, 0, 500], [1, 598, 1], [0, 300, 129]):
        for x in (q, k, v):
            x.copy_(randn(g, *x.shape))
        start.copy_(starts(lengths))
        out.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        used = sum(lengths)
        ref, tol = prompt_ref(q, k, v, lengths, heads, kv, dim, 0.1)
        within(out[:used], ref, tol)
        assert (out[used:] == 3).all()
    assert status() == 0


def test_prompt_bad_extents_are_left_out_and_reported():
    g = gen(25)
    heads = kv = 2
    dim, T = 64, 50
    q, k, v = (randn(g, T, heads * dim, dtype=F16) for _ in range(3))
    for start in ([0, 20, 51], [0, 20, 10], [0, 20, 2 ** 31 - 1]):
        out = torch.full((T, heads * dim), 3.0, dtype=F16, device="cuda")
        prompt(q, k, v, i32(start), heads, kv, dim, 0.1, out=out)
        assert status() == 4 and status() == 0
        ref, tol = prompt_ref(q, k, v, [20], heads, kv, dim, 0.1)
        within(out[:20], ref, tol)
        assert (out[20:] == 3).all()


# ---------------------------------------------------------------------------------- together

@pytest.mark.parametrize("page,heads,kv,dim,pairs", [(16, 9, 3, 64, 1), (64, 20, 5, 128, 0)])
def test_a_prompt_and_its_steps(page, heads, kv, dim, pairs):
    """As a serving loop runs them: packed prompts are appended and attended to, then steps of one token
    each, the step captured once as a graph on a side stream and replayed with positions that it
    advances itself.  Each result is held to 64 bits over the cache as it stands."""
    g = gen(31)
    lengths, steps = [37, 1, 150], 20
    S, T, scale = len(lengths), sum(lengths), dim ** -0.5
    total, table = tables(g, [n + steps for n in lengths], page)
    table = i32([r[:-2] + [0, 0] for r in table])
    c = Cache(total, page, kv, dim)
    rope = torch.from_numpy(rope_table(256, dim)).cuda()
    x = randn(g, T, (heads + 2 * kv) * dim)
    q, k, v = x.split([heads * dim, kv * dim, kv * dim], 1)
    qo, ko, vo = (torch.empty(T, n * dim, dtype=F16, device="cuda") for n in (heads, kv, kv))
    zero = i32([0] * S)
    append(c, append_args(q, k, v, starts(lengths), zero, table, rope, dim, pairs, F16, qo, ko, vo, heads=heads))
    out = prompt(qo, ko, vo, starts(lengths), heads, kv, dim, scale, out_type=F32)
    ref, tol = prompt_ref(qo, ko, vo, lengths, heads, kv, dim, scale)
    within(out, ref, tol)

    pos, one = i32(lengths), i32([1] * S)
    start = i32(list(range(S + 1)))
    x = torch.empty(S, (heads + 2 * kv) * dim, device="cuda")
    q, k, v = x.split([heads * dim, kv * dim, kv * dim], 1)
    qo = torch.empty(S, heads * dim, device="cuda")
    out = torch.empty(S, heads * dim, device="cuda")
    ws = workspace(S, heads, c)
    length = pos.clone()

    def step():
        length.copy_(pos + one)
        append(c, append_args(q, k, v, start, pos, table, rope, dim, pairs, F32, qo, heads=heads))
        decode(c, qo, length, table, heads, scale, ws=ws, out=out)
        pos.add_(one)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.copy_(randn(g, *x.shape))
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(1, steps):
        x.copy_(randn(g, *x.shape))
        graph.replay()
        torch.cuda.synchronize()
        now = [n + i + 1 for n in lengths]
        assert length.tolist() == now
        ref, tol = decode_ref(c, qo, now, table, heads, scale)
        within(out, ref, tol)
    assert status() == 0
