"""Calls of the token stage's operators that their documentation allows and that once went wrong, on the GPU against
oracle/token_stage_ref.py."""
import math

import numpy as np
import pytest
import torch

from oracle import token_stage_ref as ref
from pigeon_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _ids(x, u, temperature, k, p, q):
    """The oracle's ids, with the numbers as the fp32 that the call makes of them."""
    f32 = lambda v: float(np.float32(v))                            # noqa: E731
    xn, un = x.cpu().double().numpy(), u.cpu().double().numpy()
    return [ref.sample_tokens_ref(xn[b], un[b], f32(temperature), k, f32(p), f32(q)) for b in range(len(xn))]


# ------------------------------------------------------------------------------------------------ top-k at a full list
LIST = 4096                                                         # ids that the kernel sorts


def _border(row, temperature, k):
    """Of the bins over the distance to the maximum, 32 to a factor of two of weight, in fp32 as the kernel places
    them: ids before the bin that holds rank k, ids in it, and the ids from its lower end with 1 % of a bin of slack."""
    x, f32 = row.cpu().float().numpy(), np.float32
    fc = f32(32 * 1.44269504088896340736 / float(f32(temperature)))
    bins = np.minimum(np.maximum((x.max() - x) * fc, f32(0)), f32(2047)).astype(np.int64)
    count = np.bincount(bins, minlength=2048)
    upto = count.cumsum()
    cut = int(np.searchsorted(upto, k))
    low = f32(float(x.max()) - (cut + 1.01) / float(fc))
    return int(upto[cut] - count[cut]), int(count[cut]), int((x >= low - abs(low) * f32(2.0 ** -23)).sum())


def _two_levels(V, many, dt):
    """`many` ids at 2.5 and the others 1/64 under it, which is 1.0019 bins at a temperature of 0.72."""
    x = torch.full((4, V), 2.5 - 1.0 / 64)
    x[:, V // 7:V // 7 + many] = 2.5
    return x.to(dt).to(DEV)


@pytest.mark.parametrize("filters", [(1.0, 0.0), (0.9, 0.0), (0.97, 0.3)])
@pytest.mark.parametrize("case", ["normal", "levels", "few levels", "levels fp32"])
def test_top_k_where_ids_just_behind_the_border_would_overfill_the_list(case, filters):
    """The bins up to the border fit the list and the ids near its lower end do not: the pass over all ids, which is the
    last, has to take the former alone."""
    if case == "normal":
        g = torch.Generator().manual_seed(1)
        x = (torch.randn(131072, generator=g) * 0.5).to(torch.bfloat16).expand(4, -1).contiguous().to(DEV)
        temperature, ks = 1.18, (3644, 3900, 4057)
    else:
        x = _two_levels(5000 if case == "few levels" else 48386, 3000, torch.float32 if case == "levels fp32" else torch.bfloat16)
        temperature, ks = 0.72, (50, 1000, 1025, 2999, 3000)
    u = torch.tensor([0.0, 0.3, 0.71, 0.9999], device=DEV)
    p, q = filters
    for k in ks:
        before, inside, near = _border(x[0], temperature, k)
        assert before + inside <= LIST < near, (before, inside, near)        # the state in question
        got = ops.sample_tokens(x, u, temperature=temperature, top_k=k, top_p=p, min_p=q)
        assert got.tolist() == _ids(x, u, temperature, k, p, q), (case, k)


@pytest.mark.parametrize("many", [4095, 4096, 4097])
def test_top_k_with_as_many_ids_as_the_list_takes(many):
    """Both sides of the list's length, the border in its last bin and behind it."""
    x, u = _two_levels(30000, many, torch.bfloat16), torch.tensor([0.0, 0.5, 0.8, 0.9999], device=DEV)
    for k in (40, 1025, many - 1, many, many + 1, 9000):
        for p in (1.0, 0.8):
            assert ops.sample_tokens(x, u, temperature=0.72, top_k=k, top_p=p).tolist() == _ids(x, u, 0.72, k, p, 0.0), (k, p)


# ------------------------------------------------------------------------------------------------ min-p above every weight
@pytest.mark.parametrize("min_p", [0.5, 1.0, 1.5, 2.0, math.inf, math.nan])
@pytest.mark.parametrize("temperature", [math.inf, 3e38, 1.0])
@pytest.mark.parametrize("V,top_k", [(4, 0), (4, 3), (3001, 0), (3001, 40), (3001, 900), (40000, 0), (40000, 5000), (48386, 4000)])
def test_min_p_leaves_the_same_ids_in_the_sums_and_in_the_draw(V, top_k, temperature, min_p):
    """At a high temperature weights of ids under the maximum are 1 too: above 1, or NaN, min-p leaves the largest logits
    alone, at 1 and below all of them.  Sums over more than the draw finds leave an id unwritten."""
    x = -(torch.arange(V) % 1000).float() / 64
    x = torch.stack([x, x.flip(0), torch.zeros(V), x.roll(V // 3)])
    x[1, V // 2] = -math.inf
    u = torch.tensor([0.9, 0.0, 0.6, 0.9999], device=DEV)
    for dt in (torch.float32, torch.bfloat16):
        y = x.to(dt).to(DEV)
        for p in (1.0, 0.75):
            want = _ids(y, u, temperature, top_k, p, min_p)
            assert ops.sample_tokens(y, u, temperature=temperature, top_k=top_k, top_p=p, min_p=min_p).tolist() == want, (dt, p)
            rows = torch.full((4,), min_p, device=DEV)
            assert ops.sample_tokens(y, u, temperature=temperature, top_k=top_k, top_p=p, min_p=rows).tolist() == want, (dt, p)


# ------------------------------------------------------------------------------------------------ attention: layouts of q
def _attention_inputs(T, H, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    P, N = 16, 12
    cache = [torch.randn(N, H, P, D, generator=g).to(torch.float8_e4m3fn).to(DEV), torch.randn(N, H, D, P, generator=g).to(torch.float8_e4m3fn).to(DEV),
             torch.ones(N, H, device=DEV), torch.ones(N, H, device=DEV)]
    table = torch.randperm(N, generator=g)[:4 * min(T, 3)].view(-1, 4).to(torch.int32).to(DEV)
    return cache, table, torch.full((len(table),), 61, dtype=torch.int32, device=DEV), g


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,Hq,D", [(1, 4, 64), (3, 1, 128), (1, 1, 64), (1, 2, 256)])
@pytest.mark.parametrize("pitch,first", [(3, 0), (3, 2), (8, 8), (8, 4), (0, 1)])
def test_queries_of_one_token_or_one_head_with_any_stride(T, Hq, D, pitch, first, dt):
    """Slices of wider rows: torch calls a tensor contiguous whatever the stride of an axis of length 1 is."""
    cache, table, lens, g = _attention_inputs(T, 1, D)
    if T == 1:                                                      # a row of a [2, heads, D] tensor
        q = torch.randn(2, Hq * D + pitch + first, generator=g).to(dt).to(DEV)[:, first:first + Hq * D].unflatten(1, (Hq, D))[:1]
        assert q.is_contiguous() and q.stride(0) == Hq * D + pitch + first
    else:                                                           # a head of a [2, T, D] tensor
        q = torch.randn(2, T * D + pitch + first, generator=g).to(dt).to(DEV)[:, first:first + T * D].unflatten(1, (T, D)).transpose(0, 1)[:, :1]
        assert q.is_contiguous() and q.stride(1) == T * D + pitch + first
    starts = None if T == len(lens) else torch.tensor([0, T], dtype=torch.int32, device=DEV)
    plain = torch.empty(T, Hq, D, dtype=dt, device=DEV)
    plain.copy_(q)
    want = ops.cached_attention(plain, *cache, table, lens, starts=starts)
    assert torch.equal(ops.cached_attention(q, *cache, table, lens, starts=starts), want)
    out = torch.empty(T, Hq, D + 3, dtype=dt, device=DEV)[:, :, 1:D + 1]
    assert torch.equal(ops.cached_attention(q, *cache, table, lens, starts=starts, out=out), want)


# ------------------------------------------------------------------------------------------------ refusals
def test_tables_without_a_column_and_caches_without_a_page_are_refused_by_name():
    cache, table, lens, g = _attention_inputs(2, 1, 64)
    q = torch.randn(2, 1, 64, generator=g).to(torch.bfloat16).to(DEV)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)                               # noqa: E731
    empty = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="column"):
        ops.cached_attention(q, *cache, empty, i32(2))
    with pytest.raises(ValueError, match="column"):
        ops.page_advance(i32(2), i32(2), empty, i32(4), i32(1), 16, 2)
    with pytest.raises(ValueError, match="room for a page"):
        ops.page_advance(i32(2), i32(2), table, i32(0), i32(1), 16, 2)
    none = [t[:0] for t in cache]
    with pytest.raises(ValueError, match="page and a head"):
        ops.cached_attention(q, *none, table, lens)
    with pytest.raises(ValueError, match="page and a head"):
        ops.cache_write(q, q, torch.zeros(2, dtype=torch.int64, device=DEV), *none)
    # nothing to do is no error, whatever there is to do it with
    assert ops.cached_attention(q, *cache, empty[:0], i32(0), starts=i32(1)).shape == q.shape
    assert ops.cached_attention(q[:0], *none, empty, i32(2), starts=i32(3)).shape == (0, 1, 64)
    ops.cache_write(q[:0], q[:0], torch.zeros(0, dtype=torch.int64, device=DEV), *none)
    assert ops.page_advance(i32(0), i32(0), empty[:0], i32(0), i32(1), 16, 2)["slots"].tolist() == [-1, -1]


def test_sizes_that_would_be_cut_to_32_bits_are_refused():
    """2^32 + n must not pass for n, nor -2^32 + n."""
    cache, table, lens, g = _attention_inputs(2, 1, 64)
    q = torch.randn(2, 1, 64, generator=g).to(torch.bfloat16).to(DEV)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)                               # noqa: E731
    for window in (-1, -2 ** 31, -2 ** 32, -2 ** 32 + 5):
        with pytest.raises(ValueError):
            ops.cached_attention(q, *cache, table, lens, window=window)
    for page_size in (2 ** 32 + 16, -2 ** 32 + 64, 2 ** 31, 0, -16):
        with pytest.raises(NotImplementedError):
            ops.page_advance(i32(2), i32(2), table, i32(4), i32(1), page_size, 2)


def test_an_output_whose_rows_are_one_is_refused():
    cache, table, lens, g = _attention_inputs(3, 1, 64)
    q = torch.randn(3, 2, 64, generator=g).to(torch.bfloat16).to(DEV)
    for out in (q[:1].clone().expand(3, 2, 64), q[:, :1].clone().expand(3, 2, 64)):
        with pytest.raises(ValueError, match="out"):
            ops.cached_attention(q, *cache, table, lens, out=out)
    one = q[:1, :1].clone()                                         # an axis of length 1 may have any stride
    got = ops.cached_attention(q[:1, :1], *cache, table[:1], lens[:1], out=one.as_strided((1, 1, 64), (0, 0, 1)))
    assert torch.equal(got, ops.cached_attention(q[:1, :1].contiguous(), *cache, table[:1], lens[:1]))
    turned = torch.empty(2, 3, 64, dtype=q.dtype, device=DEV).transpose(0, 1)                   # heads before tokens
    assert torch.equal(ops.cached_attention(q, *cache, table, lens, out=turned), ops.cached_attention(q, *cache, table, lens))
    same = q.clone()                                                # in place of the queries
    assert torch.equal(ops.cached_attention(same, *cache, table, lens, out=same), ops.cached_attention(q, *cache, table, lens))


# ------------------------------------------------------------------------------------------------ two at once
def test_calls_on_two_streams_at_once_keep_apart():
    """Split attention, top-p sampling and the bookkeeping of two batches side by side: each call has its own workspace."""
    g = torch.Generator().manual_seed(5)
    P, D, H, W = 64, 128, 2, 150
    batches = []
    for R in (1, 3):
        N = R * W + 4
        cache = [torch.randn(N, H, P, D, generator=g).to(torch.float8_e4m3fn).to(DEV), torch.randn(N, H, D, P, generator=g).to(torch.float8_e4m3fn).to(DEV),
                 torch.ones(N, H, device=DEV), torch.ones(N, H, device=DEV)]
        table = torch.randperm(N, generator=g)[:R * W].view(R, W).to(torch.int32).to(DEV)
        lens = torch.randint(5000, W * P - 1, (R,), generator=g, dtype=torch.int32).to(DEV)
        q = torch.randn(R, 4 * H, D, generator=g).to(torch.bfloat16).to(DEV)
        logits, u = torch.randn(R, 60000, generator=g).to(DEV) * 2, torch.rand(R, generator=g).to(DEV)
        batches.append((cache, table, lens, q, logits, u, torch.arange(N, dtype=torch.int32, device=DEV)))

    def step(b):
        cache, table, lens, q, logits, u, pool = b
        held, t, free, count = lens.clone(), table.clone(), pool.clone(), torch.full((1,), 4, dtype=torch.int32, device=DEV)
        plan = ops.page_advance(held, torch.ones_like(held), t, free, count, P, len(held))
        return ops.cached_attention(q, *cache, table, lens), ops.sample_tokens(logits, u, top_p=0.95), plan["slots"], held, t
    want = [step(b) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(batches[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
