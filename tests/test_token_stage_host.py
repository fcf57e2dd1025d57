"""Host side of the token stage's operators, without a GPU: what the C entry points refuse before any launch, workspace
sizes, and the oracle's own rules."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import token_stage_ref as ref
from pigeon_amd import _lib, ops


def _p16():
    buf = ctypes.create_string_buffer(64)
    return (ctypes.addressof(buf) + 15) & ~15, buf


def test_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    p, _keep = _p16()
    adv = lambda **k: lib.pgn_page_advance(*[{**dict(lens=p, keep=None, add=p, table=p, ts=4, free=p, count=p, N=4, R=2, W=4, P=16, T=8,       # noqa: E731
                                                     slots=p, starts=p, status=p, stream=None), **k}[n] for n in
                                             ("lens", "keep", "add", "table", "ts", "free", "count", "N", "R", "W", "P", "T", "slots", "starts", "status", "stream")])
    for k in ("lens", "add", "table", "free", "count", "slots", "starts", "status"):
        assert adv(**{k: None}) == -1, k
    for k in ({"R": 0}, {"W": 0}, {"N": 0}, {"T": -1}, {"ts": 3}, {"R": -1}):
        assert adv(**k) == -1, k
    for k in ({"P": 24}, {"P": 0}, {"P": 256}, {"T": 1 << 31}, {"W": 1 << 28, "ts": 1 << 28}):
        assert adv(**k) == -2, k

    wr = lambda **k: lib.pgn_cache_write(*[{**dict(k=p, v=p, dt=1, slots=p, T=2, H=2, D=64, kst=128, ksh=64, vst=128, vsh=64, kp=p, vp=p,       # noqa: E731
                                                   ks=p, vs=p, N=4, P=16, stream=None), **k}[n] for n in
                                           ("k", "v", "dt", "slots", "T", "H", "D", "kst", "ksh", "vst", "vsh", "kp", "vp", "ks", "vs", "N", "P", "stream")])
    for k in ("k", "v", "slots", "kp", "vp", "ks", "vs"):
        assert wr(**{k: None}) == -1, k
    for k in ({"T": 0}, {"H": 0}, {"D": 0}, {"N": 0}, {"k": p + 1}, {"kp": p + 8}, {"vp": p + 4}):
        assert wr(**k) == -1, k
    for k in ({"dt": 0}, {"dt": 7}, {"D": 80}, {"P": 8}, {"H": 70000}, {"T": 1 << 31}):
        assert wr(**k) == -2, k

    names = ("q", "dt", "kp", "vp", "ks", "vs", "table", "ts", "lens", "starts", "out", "T", "R", "Hq", "Hkv", "D", "N", "W", "P", "qst", "qsh", "ost",
             "osh", "scale", "causal", "window", "ws", "wsb", "stream")
    base = dict(q=p, dt=1, kp=p, vp=p, ks=p, vs=p, table=p, ts=4, lens=p, starts=p, out=p, T=2, R=2, Hq=4, Hkv=2, D=64, N=4, W=4, P=16, qst=256,
                qsh=64, ost=256, osh=64, scale=0.1, causal=1, window=0, ws=None, wsb=0, stream=None)
    att = lambda **k: lib.pgn_cached_attention(*[{**base, **k}[n] for n in names])                                                            # noqa: E731
    for k in ("q", "kp", "vp", "ks", "vs", "table", "lens", "out"):
        assert att(**{k: None}) == -1, k
    for k in ({"T": 0}, {"R": 0}, {"Hq": 3}, {"Hkv": 0}, {"N": 0}, {"W": 0}, {"ts": 3}, {"window": -1}, {"window": 2, "causal": 0}, {"scale": float("nan")},
              {"starts": None, "T": 3}, {"q": p + 2}, {"qst": 250}, {"qsh": 60}, {"kp": p + 8}, {"out": p + 1}):
        assert att(**k) == -1, k
    for k in ({"dt": 0}, {"D": 80}, {"D": 32}, {"P": 20}, {"W": 1 << 28, "ts": 1 << 28}, {"Hq": 140000, "Hkv": 70000}, {"T": 1 << 30, "Hq": 64}):
        assert att(**k) == -2, k
    # a call whose workspace is too small, misaligned or missing
    need = lib.pgn_cached_attention_workspace_bytes(1, 1, 0, 2, 2, 64, 512, 16)
    assert need > 0
    big = dict(T=1, R=1, Hq=2, Hkv=2, W=512, ts=512, starts=None)
    for k in ({"ws": None, "wsb": need}, {"ws": p, "wsb": need - 1}, {"ws": p + 8, "wsb": need}):
        assert att(**big, **k) == -1, k

    sa = lambda **k: lib.pgn_sample_tokens(*[{**dict(x=p, dt=0, st=100, B=2, V=100, u=p, t=None, ta=1.0, k=None, ka=0, pp=None, pa=1.0, m=None,  # noqa: E731
                                                     ma=0.0, ids=p, stream=None), **k}[n] for n in
                                             ("x", "dt", "st", "B", "V", "u", "t", "ta", "k", "ka", "pp", "pa", "m", "ma", "ids", "stream")])
    for k in ({"x": None}, {"u": None}, {"ids": None}, {"B": 0}, {"V": 0}, {"st": -100}, {"x": p + 2}, {"dt": 1, "x": p + 1}):
        assert sa(**k) == -1, k
    for k in ({"dt": 5}, {"V": 262145, "st": 262145}):
        assert sa(**k) == -2, k


def test_attention_refuses_tables_beyond_the_positions_it_counts():
    """W * P up to PGN_CACHED_MAX_KEYS passes the check of sizes (here it fails for its missing workspace, before any launch)."""
    lib = _lib.load()
    p, _keep = _p16()
    call = lambda W, P: lib.pgn_cached_attention(p, 1, p, p, p, p, p, W, p, p, p, 2, 2, 4, 2, 64, 4, W, P, 256, 64, 256, 64, 0.1, 1, 0, None, 0,   # noqa: E731
                                                 None)
    for P in (16, 32, 64, 128):
        assert call((1 << 28) // P, P) == -1 and call((1 << 28) // P + 1, P) == -2


def test_workspace_is_zero_or_whole_and_grows_with_the_splits():
    f = _lib.load().pgn_cached_attention_workspace_bytes
    assert f(0, 1, 0, 1, 1, 64, 1, 16) == 0 and f(1, 1, 0, 3, 2, 64, 1, 16) == 0
    assert f(512, 512, 0, 32, 32, 128, 256, 16) == 0                 # enough workgroups without splitting
    for W in (1, 16, 17, 200, 8192):
        n = f(1, 1, 0, 8, 8, 128, W, 16)
        assert n % (8 * (128 * 4 + 8)) == 0


def test_workspace_does_not_grow_with_the_tokens_of_long_prompts():
    """Few requests split their keys over many workgroups, but only as long as there are few rows: at most 512 workgroups
    of 64 rows, and twice 512 of 128, each with head_dim + 2 numbers a row."""
    f = _lib.load().pgn_cached_attention_workspace_bytes
    for R in (1, 3, 40):
        for T in (64, 1000, 8192, 100000, 1000000):
            for Hq, Hkv in ((32, 32), (32, 8), (16, 1)):
                for W in (16, 8192, 200000):
                    assert f(T, R, 1, Hq, Hkv, 128, W, 16) <= (2 * 512 * 64 + 2 * 512 * 128) * (128 * 4 + 8), (R, T, Hq, Hkv, W)


def test_cpu_tensors_raise():
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.page_advance(z, z, torch.zeros(2, 2, dtype=torch.int32), z, z[:1], 16, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.sample_tokens(torch.zeros(2, 5), torch.zeros(2))
    c = [torch.zeros(1, 1, 16, 64).to(torch.float8_e4m3fn), torch.zeros(1, 1, 64, 16).to(torch.float8_e4m3fn), torch.ones(1, 1), torch.ones(1, 1)]
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.cached_attention(torch.zeros(2, 1, 64, dtype=torch.bfloat16), *c, torch.zeros(2, 1, dtype=torch.int32), z)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.cache_write(torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64), *c)


def test_oracle_e4m3_equals_torchs_conversion():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.linspace(-0.05, 0.05, 20001), torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0])])
    assert np.array_equal(ref.e4m3_round(x.numpy()), x.to(torch.float8_e4m3fn).double().numpy())
    assert ref.page_scale(448.0) == 1.0 and ref.page_scale(448.1) == 2.0 and ref.page_scale(224.0) == 0.5 and ref.page_scale(0.0) == 2.0 ** -100


def test_oracle_attention_with_pages_that_are_none():
    """A bad page hides its keys: the same as a request without them."""
    g = torch.Generator().manual_seed(0)
    kp = torch.randn(4, 1, 16, 64, generator=g).to(torch.float8_e4m3fn)
    vp = torch.randn(4, 1, 64, 16, generator=g).to(torch.float8_e4m3fn)
    one = torch.ones(4, 1)
    q = torch.randn(1, 1, 64, generator=g).to(torch.bfloat16)
    a = ref.cached_attention_ref(q, kp, vp, one, one, torch.tensor([[0, 9, 2]]), torch.tensor([40]))[0]
    b = ref.cached_attention_ref(q, kp, vp, one, one, torch.tensor([[0, 2]]), torch.tensor([24]))[0]
    assert torch.equal(a, b)
    c = ref.cached_attention_ref(q, kp, vp, one, one, torch.tensor([[-1, 4, 77]]), torch.tensor([40]))[0]
    assert bool((c == 0).all())
