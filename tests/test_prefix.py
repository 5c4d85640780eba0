"""prefix_attention against its definition in float64, row by row over the keys that
the row sees: every shape of workgroup and head width, chunks and their joins,
lengths from none to many, windows, grouped heads; caches of any strides; what
lies behind a length or in a later token; streams and graph capture; and what it
refuses.

Tolerances.  With e = 2^-24 a score is off by at most e (D A + 2 |s| + 16), A the
sum of |q k| scaled (one product sum, its scaling, the exponential), and sums over
n keys by n e relative to the sum of magnitudes; d stands for both.  16-bit types
round each probability to their own type, by u = eps / 2 (fp16 below 2^-14 by
2^-25 at most, against a largest one of at least 1).  So an output is off by at
most (u + 4 d) times the mean of |v| (plus n 2^-25 max|v| in fp16), and half a step
of its type; the LSE by 4 d + 4 e (1 + |lse|).
"""

import math

import pytest
import torch

from _helpers import DEV, randn

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0 ** -24


def _make(case, dtype, seed=0, std=1.5):
    B, L, H, Hk, D, N, S, lens, window = case
    t = dict(q=randn((B, L, H, D), dtype, seed, std), pk=randn((N, Hk, D), dtype, seed + 1),
             pv=randn((N, Hk, D), dtype, seed + 2), k=None, v=None, lens=None, window=window)
    if S is not None:
        t["k"], t["v"] = randn((B, S, Hk, D), dtype, seed + 3), randn((B, S, Hk, D), dtype, seed + 4)
        if lens is not None:
            t["lens"] = torch.tensor([lens[b % len(lens)] for b in range(B)], dtype=torch.int32)
    return t


def _reference(t, scale=None):
    """(out, tolerance), (lse, tolerance), each row over its own keys."""
    q = t["q"].double()
    B, L, H, D = q.shape
    Hk = t["pk"].shape[1]
    scale = D ** -0.5 if scale is None else scale
    fi = torch.finfo(t["q"].dtype)
    u = 0.0 if t["q"].dtype == F32 else fi.eps / 2
    out, lse = torch.zeros_like(q), torch.full(q.shape[:-1], -math.inf, dtype=torch.float64)
    to, tl = torch.zeros_like(q), torch.zeros_like(lse)
    for b in range(B):
        n = 0 if t["k"] is None else t["k"].shape[1] if t["lens"] is None else int(t["lens"][b])
        for j in range(L):
            at = n - L + j
            lo = 0 if t["window"] is None else max(0, at - t["window"] + 1)
            ks, vs = [t["pk"].double()], [t["pv"].double()]
            if at >= 0:
                ks.append(t["k"][b, lo:at + 1].double())
                vs.append(t["v"][b, lo:at + 1].double())
            kk, vv = torch.cat(ks), torch.cat(vs)
            if kk.shape[0] == 0:
                continue
            kk, vv = (x.repeat_interleave(H // Hk, 1).transpose(0, 1) for x in (kk, vv))  # [H, n, D]
            qq = q[b, j].unsqueeze(1)
            s = (qq * kk).sum(-1) * scale
            a = (qq.abs() * kk.abs()).sum(-1).amax(-1) * scale
            l = torch.logsumexp(s, -1)
            p = torch.exp(s - l.unsqueeze(-1))
            out[b, j] = (p.unsqueeze(-1) * vv).sum(1)
            lse[b, j] = l
            d = E * (D * a + 2 * s.abs().amax(-1) + 16 + kk.shape[1])
            mean = (p.unsqueeze(-1) * vv.abs()).sum(1)
            to[b, j] = (u + 4 * d.unsqueeze(-1)) * mean + out[b, j].abs() * fi.eps / 2 + fi.tiny
            if t["q"].dtype == F16:
                to[b, j] += kk.shape[1] * 2.0 ** -25 * vv.abs().amax(1)
            tl[b, j] = 4 * d + 4 * E * (1 + l.abs())
    return (out, to), (lse, tl)


def _near(got, want, what):
    v, tol = want
    o = got.detach().cpu().double()
    assert o.shape == v.shape, what
    fin = v.isfinite()
    assert torch.equal(o.isfinite(), fin), f"{what}: finite pattern"
    assert torch.equal(o.isnan(), v.isnan()) and torch.equal(o[v.isinf()], v[v.isinf()]), what
    bad = ~((o - v).abs() <= tol)[fin]
    assert not bad.any(), (f"{what}: {int(bad.sum())}/{o.numel()} off, worst "
                           f"{float(((o - v).abs() - tol)[fin].max()):.3e} beyond")


def _run(t, **kw):
    import natten_amd

    d = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in t.items()}
    return natten_amd.prefix_attention(d["q"], d["pk"], d["pv"], d["k"], d["v"], seq_lens=d["lens"],
                                       kernel_size=d["window"], return_lse=True, **kw)


def _check(t, what="", **kw):
    out, lse = _run(t, **kw)
    assert out.dtype == t["q"].dtype and lse.dtype == F32 and out.is_contiguous()
    ro, rl = _reference(t, kw.get("scale"))
    _near(out, ro, f"{what} out")
    _near(lse, rl, f"{what} lse")


# B, tokens, heads, kv heads, dim, prefix, own capacity, lengths, window
CASES = {
    "one of everything": (1, 1, 1, 1, 8, 1, 1, [1], None),
    "prefix only": (3, 1, 4, 2, 64, 77, None, None, None),
    "prefix only, whole batch wide": (9, 2, 8, 1, 32, 300, None, None, None),
    "own only": (2, 1, 4, 2, 64, 0, 100, [100, 37], None),
    "own only, default lengths": (2, 1, 4, 4, 32, 0, 45, None, None),
    "nothing to see": (2, 3, 2, 1, 16, 0, 9, [0, 2], None),
    "small service": (4, 1, 8, 2, 64, 301, 131, [131, 0, 1, 64], None),
    "narrow, many chunks": (1, 1, 2, 2, 40, 1500, 700, [650], None),
    "wide of 64": (8, 1, 8, 2, 128, 333, 150, [150, 0, 33, 128, 129], None),
    "wide of 128": (24, 1, 8, 1, 128, 270, 70, [70, 3, 64], None),
    "wide rows of one sample": (2, 1, 34, 1, 96, 65, 66, [66, 31], None),
    "very many heads": (1, 1, 70, 1, 72, 130, 40, [40], None),
    "256 wide, narrow": (2, 1, 6, 2, 256, 90, 50, [50, 7], None),
    "256 wide, wide": (5, 3, 8, 1, 256, 70, 50, [50, 7, 2], None),
    "200 wide": (3, 1, 4, 2, 200, 45, 40, [40, 5, 0], None),
    "tokens narrow": (3, 4, 4, 2, 64, 50, 80, [80, 4, 2], None),
    "tokens wide": (2, 9, 4, 1, 64, 50, 200, [200, 150], None),
    "tokens of several tiles": (2, 70, 4, 1, 32, 130, 333, [333, 75], None),
    "tokens longer than the cache": (2, 40, 2, 1, 32, 20, 25, [25, 10], None),
    "window of one": (3, 1, 4, 2, 64, 5, 90, [90, 1, 0], 1),
    "window": (3, 1, 4, 2, 80, 65, 400, [400, 33, 300], 129),
    "window, tokens narrow": (2, 5, 3, 1, 64, 0, 300, [300, 4], 7),
    "window, tokens wide": (2, 50, 4, 2, 64, 33, 300, [300, 60], 37),
    "window over all": (2, 3, 2, 1, 64, 10, 60, [60, 20], 5000),
    "eight waves": (40, 1, 8, 2, 128, 600, 20, [20, 0, 7], None),
    "eight waves, prefix only": (70, 2, 8, 2, 96, 333, None, None, None),
    "eight waves, tokens": (6, 30, 4, 2, 80, 900, 60, [60, 31, 5, 0], None),
    "eight waves, tokens of two tiles": (3, 100, 6, 2, 128, 700, 130, [130, 101, 40], None),
    "eight waves, window": (5, 40, 4, 1, 120, 513, 150, [150, 90, 41], 33),
    "two narrow tiles": (3, 1, 32, 1, 128, 40, 300, [300, 0, 129], None),
    "two narrow tiles, tokens": (3, 5, 8, 2, 64, 20, 400, [400, 3, 260], None),
    "two narrow tiles, window": (2, 8, 4, 1, 40, 0, 300, [300, 150], 30),
    "window, tokens of several tiles": (1, 130, 3, 1, 48, 64, 400, [390], 100),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", list(CASES))
def test_against_the_definition(case, dtype):
    _check(_make(CASES[case], dtype), f"{case} {dtype}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_chunks_of_many_tiles(dtype):
    """Enough keys in all that a chunk is several tiles per wave; compared on some
    samples, and with float32 rows of the 16-bit inputs on all."""
    B, Hk, D, N, S = 96, 4, 16, 3000, 1800
    g = torch.Generator().manual_seed(1)
    t = _make((B, 1, Hk * 2, Hk, D, N, S, None, None), dtype, 5)
    t["lens"] = torch.randint(0, S + 1, (B,), generator=g, dtype=torch.int32)
    out, lse = _run(t)
    for b in (0, 41, 95):
        one = {n: (x[b:b + 1] if n in ("q", "k", "v", "lens") else x) for n, x in t.items()}
        ro, rl = _reference(one)
        _near(out[b:b + 1], ro, f"sample {b}")
        _near(lse[b:b + 1], rl, f"sample {b} lse")
    f = {n: (x.float() if isinstance(x, torch.Tensor) and x.is_floating_point() else x) for n, x in t.items()}
    o32, l32 = _run(f)
    assert (out.float() - o32).abs().max() < 2e-2 and (lse - l32).abs().max() < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 20000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_long_prompt(dtype, window):
    """Rows that fill the chip many times over, their own keys in chunks of more than
    1024; compared at some of the tokens."""
    L, S, n = 8192, 32768, 30011
    t = _make((1, L, 8, 2, 32, 70, S, [n], window), dtype, 11)
    out, lse = _run(t)
    for j in (0, 1, 4097, L - 1):
        one = {**t, "q": t["q"][:, j:j + 1], "lens": torch.tensor([n - L + j + 1], dtype=torch.int32)}
        ro, rl = _reference(one)
        _near(out[:, j:j + 1], ro, f"token {j}")
        _near(lse[:, j:j + 1], rl, f"token {j} lse")


@pytest.mark.gpu
def test_scores_far_apart_and_scales():
    for dtype in (F32, BF16, F16):
        t = _make((2, 3, 4, 2, 64, 150, 140, [140, 70], None), dtype, 3, std=12.0)
        _check(t, "far apart")
        _check(_make((2, 1, 4, 2, 64, 150, 140, [140, 70], None), dtype, 3), "scale", scale=0.7)
    t = _make((1, 1, 2, 1, 32, 400, 300, [300], None), F32, 4)
    for n in ("pk", "k"):  # rising scores: the reference point moves in every tile
        t[n] = t[n] * torch.linspace(0, 30, t[n].shape[-3]).view(-1, 1, 1)
    _check(t, "rising")


def _poison(x, at, value):
    x = x.clone()
    x[at] = value
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", ["small service", "tokens narrow", "tokens wide", "window",
                                  "window, tokens wide", "256 wide, wide", "tokens of several tiles",
                                  "eight waves", "eight waves, tokens", "eight waves, window"])
def test_what_lies_behind_the_lengths_is_not_read(case, dtype):
    t = _make(CASES[case], dtype)
    want = _run(t)
    S = t["k"].shape[1]
    for b, n in enumerate(t["lens"].tolist()):
        t["k"][b, n:], t["v"][b, n:] = float("nan"), float("inf")
        if t["window"]:  # nor what lies before every window
            lo = max(0, n - t["q"].shape[1] - t["window"] + 1)
            t["k"][b, :lo], t["v"][b, :lo] = float("inf"), float("nan")
    assert S > min(t["lens"])
    for a, w in zip(_run(t), want):
        assert torch.equal(a, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", ["tokens narrow", "tokens wide", "window, tokens narrow",
                                  "window, tokens wide", "256 wide, wide",
                                  "eight waves, tokens of two tiles", "eight waves, window"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_tokens_that_a_row_does_not_see(case, dtype, value):
    """A token that holds infinities or NaN reaches the rows that see it alone: a
    new token not the ones before it, a token that leaves the window not the ones
    after it."""
    t = _make(CASES[case], dtype)
    n, L = int(t["lens"][0]), t["q"].shape[1]
    for at in {n - 1, n - L + 1, max(0, n - L + 2 - (t["window"] or n))}:
        p = dict(t, v=_poison(t["v"], (0, at, 0, 3), value))
        _check(p, f"v at {at}")
        if math.isnan(value):
            _check(dict(t, k=_poison(t["k"], (0, at, 0, 5), value)), f"k at {at}")


@pytest.mark.gpu
def test_special_values_that_rows_see():
    for dtype in (F32, BF16):
        t = _make(CASES["small service"], dtype)
        _check(dict(t, pv=_poison(t["pv"], (200, 1, 7), float("inf"))), "inf value")
        _check(dict(t, pv=_poison(t["pv"], (300, 0, 7), float("nan"))), "nan value")
        out, lse = _run(dict(t, pk=_poison(t["pk"], (10, 1, 7), float("nan"))))
        assert out[:, :, 4:].isnan().all() and lse[:, :, 4:].isnan().all()
        assert out[:, :, :4].isfinite().all() and lse[:, :, :4].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views(dtype):
    import natten_amd

    B, L, H, Hk, D, N, S = 3, 2, 8, 2, 64, 70, 90
    lens = torch.tensor([90, 5, 41], dtype=torch.int32, device=DEV)
    q = randn((B, L, H + 2 * Hk, D), dtype, 1).to(DEV)[:, :, :H]         # of a projection
    heads_first = randn((2, B, Hk, S, D), dtype, 2).to(DEV)
    k, v = (x.transpose(1, 2) for x in heads_first)
    packed = randn((N, 2, Hk, D), dtype, 3).to(DEV)
    pk, pv = packed[:, 0], packed[:, 1]
    big = randn((B, S + 30, Hk, D + 3), dtype, 4).to(DEV)[:, 7:7 + S, :, 1:1 + D]  # odd starts

    def run(*ts, lens=lens):
        return natten_amd.prefix_attention(*ts, seq_lens=lens, return_lse=True)

    for ts in ((q, pk, pv, k, v), (q, pk, pv, big, v), (q, pk, pv, k, big), (q, pk, pv, big[:1].expand(B, S, Hk, D), v),
               (q.transpose(0, -1).contiguous().transpose(0, -1), pk, pv, k, v)):
        want = run(*(t.contiguous() for t in ts))
        for a, w in zip(run(*ts), want):
            assert torch.equal(a, w)
    want = run(q, pk, pv, k, v)
    for form in (lens.long(), lens.cpu(), lens.cpu().long(), torch.stack((lens, lens), 1)[:, 0]):
        assert torch.equal(run(q, pk, pv, k, v, lens=form)[0], want[0])
    wild = torch.tensor([1 << 30, 5, 41], device=DEV)  # clamped on the device
    assert torch.equal(run(q, pk, pv, k, v, lens=wild)[0], want[0])
    wild = torch.tensor([(1 << 40), 5, 41], device=DEV)
    assert torch.equal(run(q, pk, pv, k, v, lens=wild)[0], want[0])
    none = run(q, pk, pv, k, v, lens=torch.tensor([-5, 5, 41], device=DEV, dtype=torch.int32))
    assert torch.equal(none[0], run(q, pk, pv, k, v, lens=torch.tensor([0, 5, 41], device=DEV))[0])


@pytest.mark.gpu
def test_empty_calls():
    import natten_amd

    for B, L in ((0, 1), (2, 0)):
        t = _make((B, L, 4, 2, 32, 5, 6, [3], None), BF16)
        out, lse = _run(t)
        assert out.shape == (B, L, 4, 32) and lse.shape == (B, L, 4)
    q = randn((2, 1, 4, 32)).to(DEV)
    none = torch.empty(0, 2, 32, device=DEV)
    out, lse = natten_amd.prefix_attention(q, none, none, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    cache = torch.empty(2, 0, 2, 32, device=DEV)
    out, lse = natten_amd.prefix_attention(q, none, none, cache, cache, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    assert torch.equal(natten_amd.prefix_attention(q, none, none), out)


@pytest.mark.gpu
def test_against_causal_neighborhood_attention():
    """The last rows of na1d, causal, with the prefix as additional tokens; and the
    same from its two parts by merge_attentions."""
    import natten_amd

    B, T, H, Hk, D, N, W, L = 2, 150, 4, 2, 64, 40, 31, 6
    q, k, v = randn((B, T, H, D), F32, 1).to(DEV), *(randn((B, T, Hk, D), F32, s).to(DEV) for s in (2, 3))
    pk, pv = (randn((N, Hk, D), F32, s).to(DEV) for s in (4, 5))
    ex = [t.expand(B, N, Hk, D) for t in (pk, pv)]
    want, wl = natten_amd.na1d(q, k, v, kernel_size=W, is_causal=True, return_lse=True,
                               additional_keys=ex[0], additional_values=ex[1])
    got, gl = natten_amd.prefix_attention(q[:, -L:], pk, pv, k, v, kernel_size=W, return_lse=True)
    assert torch.allclose(got, want[:, -L:], rtol=1e-5, atol=1e-5)
    assert torch.allclose(gl, wl[:, -L:], rtol=1e-5, atol=1e-5)
    a, la = natten_amd.prefix_attention(q, pk, pv, return_lse=True)
    b, lb = natten_amd.na1d(q, k, v, kernel_size=W, is_causal=True, return_lse=True)
    merged, ml = natten_amd.merge_attentions([a, b], [la, lb])
    assert torch.allclose(merged, want, rtol=1e-5, atol=1e-5)
    assert torch.allclose(ml, wl, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_streams_twin_and_capture():
    import natten_amd
    import natten_amd.autograd.fused as AF

    t = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x
         for n, x in _make(CASES["wide of 64"], BF16).items()}

    def step():
        return natten_amd.prefix_attention(t["q"], t["pk"], t["pv"], t["k"], t["v"],
                                           seq_lens=t["lens"], return_lse=True)

    want = step()
    with AF.python_autograd():
        twin = step()
    side, second = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    second.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(second):  # two calls at once, each with its own workspace
        beside = step()
    graphs, helds = [], []
    with torch.cuda.stream(side):
        other = step()
        torch.cuda.synchronize()
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                helds.append(step())
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c, d in zip(want, twin, other, beside):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)
    for r in range(3):
        t["lens"].copy_(torch.tensor([(17 * r + 31 * b) % 151 for b in range(8)]))
        t["q"].copy_(randn(t["q"].shape, BF16, 40 + r))
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for held in helds:
            for a, b in zip(step(), held):
                assert torch.equal(a, b), r


@pytest.mark.gpu
def test_refuses_to_lose_gradients():
    import natten_amd
    import natten_amd.autograd.fused as AF

    t = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x
         for n, x in _make(CASES["small service"], BF16).items()}
    for n in ("q", "pk", "pv", "k", "v"):
        d = dict(t, **{n: t[n].detach().clone().requires_grad_(True)})
        for twin in (False, True):
            with AF.python_autograd(twin):
                with pytest.raises(RuntimeError, match="no backward"):
                    natten_amd.prefix_attention(d["q"], d["pk"], d["pv"], d["k"], d["v"], d["lens"])
                with torch.no_grad():
                    natten_amd.prefix_attention(d["q"], d["pk"], d["pv"], d["k"], d["v"], d["lens"])
    with pytest.raises(ValueError, match="seq_lens must be in"):
        natten_amd.prefix_attention(t["q"], t["pk"], t["pv"], t["k"], t["v"], torch.tensor([1, 2, 3, 132]))
    with pytest.raises(RuntimeError, match="devices|HIP"):
        natten_amd.prefix_attention(t["q"], t["pk"].cpu(), t["pv"], t["k"], t["v"])


def test_refusals():
    import natten_amd
    from natten_amd._core import _lib

    q, p, k = torch.randn(2, 1, 4, 16), torch.randn(5, 2, 16), torch.randn(2, 7, 2, 16)
    n = torch.tensor([3, 4])
    with pytest.raises(RuntimeError, match="HIP"):
        natten_amd.prefix_attention(q, p, p, k, k, n)
    for args, kw, match in (
            ((q[0], p, p), {}, "query must be"),
            ((q, p, p[:4]), {}, "prefix_key and prefix_value"),
            ((q, p[..., :8], p[..., :8]), {}, "prefix_key and prefix_value"),
            ((q, p[:, :0], p[:, :0]), {}, "prefix_key and prefix_value"),
            ((q[:, :, :3], p, p), {}, "divisible"),
            ((q[..., :12], p[..., :12], p[..., :12]), {}, "multiple of 8"),
            ((torch.randn(1, 1, 1, 264), torch.randn(1, 1, 264), torch.randn(1, 1, 264)), {}, "up to 256"),
            ((q, p, p, k), {}, "both be provided"),
            ((q, p, p, k, k[:, :5]), {}, "key and value must be"),
            ((q, p, p, k[:1], k[:1]), {}, "key and value must be"),
            ((q, p, p, k[:, :, :1], k[:, :, :1]), {}, "key and value must be"),
            ((q, p.half(), p), {}, "query's dtype"),
            ((q, p, p, k, k.half()), {}, "query's dtype"),
            ((q, p, p), dict(seq_lens=n), "missing"),
            ((q, p, p, k, k), dict(seq_lens=n[:1]), "length B=2"),
            ((q, p, p, k, k), dict(seq_lens=n.float()), "int32 or int64"),
            ((q, p, p, k, k), dict(kernel_size=0), "kernel_size"),
            ((q, p, p, k, k), dict(kernel_size=2.0), "kernel_size"),
            ((q, p, p), dict(scale=0.0), "scale"),
            ((q, p, p), dict(scale=-1.0), "scale"),
            ((q, p, p), dict(scale=float("nan")), "scale")):
        with pytest.raises(ValueError, match=match):
            natten_amd.prefix_attention(*args, **kw)

    lib = _lib.load()

    def params(**kw):
        return _lib.NaPrefixParams(**{**dict(batch=2, tokens=1, heads=4, kv_heads=2, head_dim=16,
                                             dtype=2, prefix=5, capacity=7, scale=0.25), **kw})

    def rc(p):
        return lib.na_prefix_fwd(p, *([None] * 8), 0, None)

    assert rc(params()) == 1 and b"non-NULL" in lib.na_last_error()
    assert lib.na_prefix_workspace_bytes(params()) >= 2 * 4 * 2 * (16 + 2) * 4
    assert lib.na_prefix_workspace_bytes(params(capacity=0)) == 0  # one chunk: written at once
    assert rc(params(batch=0)) == 0 and rc(params(tokens=0)) == 0
    for bad in (dict(heads=3), dict(kv_heads=0), dict(dtype=5), dict(prefix=-1), dict(capacity=-1),
                dict(window=-1), dict(scale=0.0), dict(scale=math.inf), dict(scale=math.nan)):
        assert rc(params(**bad)) == 1, bad
    for bad in (dict(head_dim=12), dict(head_dim=264), dict(batch=1 << 20, tokens=1 << 9),
                dict(prefix=(1 << 30) + 1)):
        assert rc(params(**bad)) == 2, bad
