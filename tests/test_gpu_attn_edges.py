"""Calls of the attention operators that their documentation allows at its edges, against the definitions in 64 bits
(tests/attn_ref.py)."""
import numpy as np
import pytest
import torch

from attn_ref import (Cache, append, append_args, append_ref, check, decode, decode_ref, i32, prompt, prompt_ref,
                      rope_table, starts, status, within, workspace)
from project_willamette_b200 import _abi

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("page,dim,n,first", [(32, 64, 1, 5), (16, 128, 3, 15), (128, 64, 90, 20)])
def test_append_to_pages_with_negative_scales(page, dim, n, first):
    """A page that other code filled with a negative scale keeps its sign and grows by its size: what is appended
    is the mirror image of the same page with all signs turned."""
    g = gen(page)
    kv, need = 3, -(-(first + n) // page)
    c = Cache(need + 1, page, kv, dim)
    c.k.random_(-127, 128, generator=g)
    c.v.random_(-127, 128, generator=g)
    c.ks.uniform_(0.0005, 0.05, generator=g)
    c.vs.uniform_(0.0005, 0.05, generator=g)
    for size in (0.0, 0.3, 40.0):  # nothing new, values that fit, values that do not
        k, v = randn(g, n, kv * dim) * size, randn(g, n, kv * dim) * size
        rope = rope_table(first + n, 0)
        table = [list(range(need))]
        want, _, _, _ = append_ref(c, None, k, v, [n], [first], table, rope, 0, 0)
        turned = c.clone()
        for codes, scale in ((turned.k, turned.ks), (turned.v, turned.vs)):
            codes[0, 1:].neg_()  # heads 1 and 2 of the begun page
            scale[0, 1:].neg_()
        append(turned, append_args(None, k, v, starts([n]), i32([first]), i32(table), None, 0, 0, F32, heads=kv))
        torch.cuda.synchronize()
        assert status() == 0
        for got, ref in zip((turned.k, turned.ks, turned.v, turned.vs), want):
            ref = torch.from_numpy(ref).cuda()
            ref[0, 1:].neg_()
            assert torch.equal(got, ref)


@pytest.mark.parametrize("dim,dtype,out", [(64, F16, F16), (128, BF16, BF16), (128, F16, F32), (64, BF16, F32)])
def test_prompt_rows_computed_again(dim, dtype, out):
    """An infinity and a NaN in the last value row: all rows before it in its tile are computed a second time, by
    other threads than those that stored them first. What stays is the second result, every time."""
    g = gen(dim)
    heads, kv, lengths = 6, 2, [128, 300, 77]
    T = sum(lengths)
    q = randn(g, T, heads * dim, dtype=dtype)
    k, v = randn(g, T, kv * dim, dtype=dtype), randn(g, T, kv * dim, dtype=dtype)
    ref, tol = prompt_ref(q, k, v, lengths, heads, kv, dim, 0.1)
    ends = np.cumsum(lengths) - 1
    v[ends, 3], v[ends, dim + 5] = float("inf"), float("nan")
    sees = torch.zeros(T, dtype=torch.bool, device="cuda")
    sees[ends.tolist()] = True
    first = None
    for _ in range(20):
        got = prompt(q, k, v, starts(lengths), heads, kv, dim, 0.1, out_type=out)
        within(got[~sees], ref[~sees], tol[~sees])
        first = got if first is None else first
        assert torch.equal(got[~sees], first[~sees])
    assert status() == 0


@pytest.mark.parametrize("dim,dtype,scale", [(64, F16, 0.125), (128, BF16, 0.09), (128, F16, -0.2)])
def test_prompt_row_depends_on_what_it_sees_alone(dim, dtype, scale):
    """Bit for bit: a row's result stays when the other rows' queries, the keys and values that its mask leaves out
    and the neighbouring sequences change."""
    g = gen(7 * dim)
    heads, kv, n = 4, 2, 600
    q = randn(g, n, heads * dim, dtype=dtype)
    k, v = randn(g, n, kv * dim, dtype=dtype), randn(g, n, kv * dim, dtype=dtype)
    alone = prompt(q, k, v, starts([n]), heads, kv, dim, scale, out_type=F32)
    # every other query much larger, so that the running maxima of those rows climb far and often
    big = q.clone()
    big[1::2] *= 40
    got = prompt(big, k, v, starts([n]), heads, kv, dim, scale, out_type=F32)
    assert torch.equal(got[0::2], alone[0::2])
    # later keys and values other and larger; packed between two other sequences
    for keep in (n - 1, 570, 513, 512, 330, 64, 1):
        a, b = k.clone(), v.clone()
        a[keep:], b[keep:] = randn(g, n - keep, kv * dim, dtype=dtype) * 30, randn(g, n - keep, kv * dim, dtype=dtype) * 30
        x, y, z = (torch.cat([randn(g, 77, t.shape[1], dtype=dtype) * 20, t, randn(g, 200, t.shape[1], dtype=dtype) * 20])
                   for t in (q, a, b))
        got = prompt(x, y, z, starts([77, n, 200]), heads, kv, dim, scale, out_type=F32)
        assert torch.equal(got[77:77 + keep], alone[:keep])


def test_waits_that_run_out_leave_later_calls_right():
    """With the shortest limit that the library takes, calls in good order may give up in the middle, with copies
    and products in flight. They say so, and calls after them, on the same SMs, are right."""
    g = gen(41)
    page, heads, kv, dim = 64, 8, 2, 128
    lengths = [9000, 400, 3000, 12000]
    total = sum(-(-n // page) for n in lengths)
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    most = max(-(-n // page) for n in lengths)
    table = i32([[order.pop() for _ in range(-(-n // page))] + [0] * (most + (-n // page)) for n in lengths])
    c = Cache(total, page, kv, dim)
    c.k.random_(-127, 128, generator=g)
    c.v.random_(-127, 128, generator=g)
    c.ks.uniform_(0.002, 0.03, generator=g)
    c.vs.uniform_(0.002, 0.03, generator=g)
    q = randn(g, len(lengths), heads * dim)
    dref, n = decode_ref(c, q, lengths, table, heads, 0.1), i32(lengths)
    rows = [900, 128, 1500]
    x, k, v = (randn(g, sum(rows), m * dim, dtype=BF16) for m in (heads, kv, kv))
    pref = prompt_ref(x, k, v, rows, heads, kv, dim, 0.1)
    L, start = _abi.lib(), starts(rows)
    torch.cuda.synchronize()
    assert status() == 0
    for _ in range(20):
        check(L.wl_set_wait_limit_ns(1000))
        try:
            a = decode(c, q, n, table, heads, 0.1)
            b = prompt(x, k, v, start, heads, kv, dim, 0.1)
            torch.cuda.synchronize()
        finally:
            check(L.wl_set_wait_limit_ns(2_000_000_000))
        flags = status()
        assert flags in (0, 1)
        if not flags:
            within(a, *dref)
            within(b, *pref)
        within(decode(c, q, n, table, heads, 0.1, ws=workspace(len(lengths), heads, c)), *dref)
        within(prompt(x, k, v, start, heads, kv, dim, 0.1), *pref)
        assert status() == 0


def test_prompts_in_a_chain():
    """Calls of both head sizes queued one behind another, each of several rounds of CTAs, so that a call's CTAs
    come while the one before still runs: the same bits as each call by itself."""
    g = gen(42)
    calls = []
    for heads, kv, dim, rows, dtype in [(9, 3, 64, [700, 1, 300, 900, 64], F16), (8, 2, 128, [1000, 129, 2000], BF16),
                                        (20, 5, 128, [1], F16), (16, 16, 64, [513, 511, 1024], BF16)]:
        x, k, v = (randn(g, sum(rows), m * dim, dtype=dtype) for m in (heads, kv, kv))
        a = (x, k, v, starts(rows), heads, kv, dim, 0.1)
        out = prompt(*a)
        torch.cuda.synchronize()
        within(out, *prompt_ref(x, k, v, rows, heads, kv, dim, 0.1))
        calls.append((a, out, torch.empty_like(out)))
    for _ in range(30):
        for a, _, other in calls:
            prompt(*a, out=other)
    torch.cuda.synchronize()
    assert status() == 0
    for _, out, other in calls:
        assert torch.equal(out, other)


@pytest.mark.parametrize("seqs,longest,heads,kv,dim,n_rot,pairs,dtype,out", [
    (500, 12, 6, 2, 64, 64, 1, F32, F16), (500, 12, 6, 2, 64, 6, 0, F32, F32), (700, 9, 20, 5, 128, 120, 0, BF16, BF16),
    (40, 300, 5, 5, 128, 10, 1, F16, F32), (1300, 140, 1, 1, 64, 64, 0, BF16, F16),
])
def test_append_queries_of_many_tokens(seqs, longest, heads, kv, dim, n_rot, pairs, dtype, out):
    """More tokens than the GPU takes query CTAs at a time, so that one CTA rotates the queries of several: across
    short and empty sequences, past one whose position is bad, with a shorter last CTA; the last case past the
    largest number of tokens a CTA."""
    g, page, P = gen(seqs), 32, np.random.default_rng(seqs)
    lengths = P.integers(0, longest + 1, seqs)
    lengths[P.integers(0, seqs, seqs // 4)] = 0
    bad = seqs // 2
    lengths[bad] = 5
    position = P.integers(0, 2 * page, seqs)
    position[bad] = 0
    ctas = 6 * torch.cuda.get_device_properties(0).multi_processor_count
    block = min(64, -(-int(lengths.sum()) // ctas))
    lengths[-1] += lengths.sum() % block == 0
    T = int(lengths.sum())
    assert block > 1 and T % block and (seqs < 1300 or T > 64 * ctas)
    need = [-(-(a + b) // page) for a, b in zip(lengths, position)]
    order = P.permutation(sum(need)).tolist()
    table = [[order.pop() for _ in range(m)] + [0] * (max(need) - m) for m in need]
    c = Cache(sum(need), page, kv, dim, fill=9)
    c.ks.uniform_(0.001, 0.05, generator=g)
    c.vs.uniform_(0.001, 0.05, generator=g)
    rope = rope_table(int(max(lengths + position)) + 1, n_rot)
    q, k, v = (randn(g, T + 3, m * dim, dtype=dtype) for m in (heads, kv, kv))
    want, rq, rk, rv = append_ref(c, q, k, v, lengths.tolist(), position.tolist(), table, rope, n_rot, pairs)
    before = c.clone()
    outs = [torch.full((T + 3, m * dim), 7.0, dtype=out, device="cuda") for m in (heads, kv, kv)]
    given = position.copy()
    given[bad] = -1
    append(c, append_args(q, k, v, starts(lengths), i32(given.tolist()), i32(table), torch.from_numpy(rope).cuda(), n_rot,
                          pairs, out, *outs, heads=heads))
    torch.cuda.synchronize()
    assert status() == 4
    skip = table[bad][0]  # the page that the bad sequence would have written
    for got, ref, old in zip((c.k, c.ks, c.v, c.vs), want, (before.k, before.ks, before.v, before.vs)):
        ref = torch.from_numpy(ref).cuda()
        ref[skip] = old[skip]
        assert torch.equal(got, ref)
    first = int(lengths[:bad].sum())
    for got, ref in zip(outs, (rq, rk, rv)):
        ref = torch.cat([torch.from_numpy(ref.reshape(T, -1)).to(out).cuda(), torch.full_like(got[T:], 7)])
        ref[first:first + 5] = 7
        assert torch.equal(got, ref)


def test_append_outputs_beside_bad_indexes():
    """A page id out of range keeps that page out of the cache and nothing else: the tokens' rotated queries, keys
    and values are written. A bad position keeps all rows of its sequence as they were."""
    g, page, heads, kv, dim = gen(44), 16, 4, 2, 64
    lengths, table = [20, 7, 18], [[0, 1], [2, 3], [4, 5]]
    T, rope = sum(lengths), rope_table(64, dim)
    q, k, v = (randn(g, T, m * dim) for m in (heads, kv, kv))
    for bad_page, bad_position in ((True, False), (False, True)):
        c = Cache(6, page, kv, dim, fill=55)
        want, rq, rk, rv = append_ref(c, q, k, v, lengths, [0, 0, 0], table, rope, dim, 0)
        outs = [torch.full((T, m * dim), 7.0, device="cuda") for m in (heads, kv, kv)]
        given = [[0, 1], [2, 3], [4, 6 if bad_page else 5]]
        append(c, append_args(q, k, v, starts(lengths), i32([0, 64 if bad_position else 0, 0]), i32(given),
                              torch.from_numpy(rope).cuda(), dim, 0, F32, *outs, heads=heads))
        torch.cuda.synchronize()
        assert status() == 4
        out = 5 if bad_page else 2  # the page that stays as it was
        assert (c.k[out] == 55).all() and (c.v[out] == 55).all() and (c.ks[out] == 0).all()
        for got, ref in zip((c.k, c.ks, c.v, c.vs), want):
            for p in set(range(6)) - {out}:
                assert torch.equal(got[p].cpu(), torch.from_numpy(ref[p]))
        for got, ref in zip(outs, (rq, rk, rv)):
            ref = torch.from_numpy(ref.reshape(T, -1)).cuda()
            if bad_position:
                ref[20:27] = 7
            assert torch.equal(got, ref)


@pytest.mark.parametrize("lengths,heads,kv,dim,dtype", [
    ([3001], 8, 1, 64, F16), ([200, 4500], 12, 1, 128, BF16), ([8192], 2, 1, 128, F16), ([6001], 2, 2, 64, BF16),
    ([1100, 1, 2049], 32, 4, 128, BF16), ([1500], 17, 1, 128, F16),
])
def test_prompt_long_and_wide_groups(lengths, heads, kv, dim, dtype):
    g = gen(sum(lengths))
    T = sum(lengths)
    q = randn(g, T, heads * dim, dtype=dtype)
    k, v = randn(g, T, kv * dim, dtype=dtype), randn(g, T, kv * dim, dtype=dtype)
    within(prompt(q, k, v, starts(lengths), heads, kv, dim, dim ** -0.5, out_type=F32),
           *prompt_ref(q, k, v, lengths, heads, kv, dim, dim ** -0.5))


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (128, BF16)])
def test_prompt_maxima_that_rise_late(dim, dtype):
    """Long stretches of like scores, then a rise past what went before, some thousand keys in and again at the end."""
    g = gen(dim + 1)
    heads, kv, n = 2, 1, 4200
    q = randn(g, n, heads * dim, dtype=dtype) * 0.1 + 1
    k = randn(g, n, dim) * 0.1
    for at, size in ((1000, 0.1), (2500, 0.4), (2563, 0.8), (4133, 1.5)):
        k[at:] += size
    k, v = k.to(dtype), randn(g, n, dim, dtype=dtype)
    for scale in (0.5, -0.5):
        within(prompt(q, k, v, starts([n]), heads, kv, dim, scale, out_type=F32),
               *prompt_ref(q, k, v, [n], heads, kv, dim, scale))


@pytest.mark.parametrize("heads,kv,dim,dtype", [(20, 5, 128, F16), (9, 3, 64, BF16)])
def test_prompt_of_nan_takes_no_longer(heads, kv, dim, dtype):
    """A NaN key makes every row that sees it NaN, and a call with it takes the time of any other: such rows used to
    be computed again one by one, which took over a hundred times as long."""
    g = gen(43)
    T, at = 2048, 3
    q, k, v = (randn(g, T, m * dim, dtype=dtype) for m in (heads, kv, kv))
    bad = k.clone()
    bad[at] = float("nan")
    start, out = starts([T]), torch.empty(T, heads * dim, dtype=dtype, device="cuda")
    got = prompt(q, bad, v, start, heads, kv, dim, 0.1)
    assert torch.isnan(got[at:]).all()
    assert torch.equal(got[:at], prompt(q, k, v, start, heads, kv, dim, 0.1)[:at])

    def shortest(keys):
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(4):
                prompt(q, keys, v, start, heads, kv, dim, 0.1, out=out)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert shortest(bad) < 20 * shortest(k)
