"""The attention operators on the GPU against their definitions in 64 bits (tests/attn_ref.py, where the bars are derived)."""
import pytest
import torch

from tests import attn_ref as R

pytestmark = pytest.mark.gpu
BF16, F64 = torch.bfloat16, torch.float64
NAN, INF = float("nan"), float("inf")


def pages(g):
    from leapquant_amd import attn
    return attn.Pages(g["kp"], g["vp"], g["ks"], g["vs"])


def attend(g, **kw):
    from leapquant_amd import attn
    kw.setdefault("gate", g["gate"])
    attn.attend(g["q"], pages(g), g["table"], g["loc"], g["lens"], g["out"], **kw)
    return g["out"]


def rope(g, **kw):
    from leapquant_amd import attn
    attn.rope_norm(g["q"], g["k"], g["v"], g["qw"], g["kw"], g["inv_freq"], pages(g), g["table"], g["loc"], g["lens"], g["out"], **kw)
    return g["out"]


def check_attend(d, window=0, scale=None, **kw):
    out = attend(R.cuda(d), window=window, scale=scale, **kw)
    R.near(out, *R.attend(d, scale=scale, window=window))
    return out


# ---- rope_norm -------------------------------------------------------------------------------------------------------------
def check_rope(d, g=None, **kw):
    g = R.cuda(d) if g is None else g
    before = {x: g[x].clone() for x in ("kp", "vp")}
    out = rope(g, **kw)
    want, k, where = R.rope(d, **kw)
    held = ~torch.isnan(want)
    eps = 2.0 ** -17                          # of a head's largest: the pair's magnitude is at most 1.42 of it
    bar = 2.0 ** -8 * want.abs() + eps * want.abs().amax(-1, keepdim=True)
    err = (out.cpu().to(F64) - want).abs()
    assert not (err[held] > bar[held]).any(), float((err - bar)[held].max())
    assert (out.cpu()[~held] == 7).all()                      # rows that no sequence holds
    for x, vals in (("kp", k), ("vp", d["v"].to(F64))):
        got, was = g[x].cpu(), before[x].cpu()
        for t, page, place in where:
            y, w = got[page, place], vals[t]
            if d["ks"] is None:
                bar = 2.0 ** -8 * w.abs() + (eps * w.abs().amax(-1, keepdim=True) if x == "kp" else 0)
                if x == "vp":
                    assert torch.equal(y, d["v"][t])
                assert not ((y.to(F64) - w).abs() > bar).any()
            else:                                             # half a step of the codes, a scale's own rounding, the eps above
                s = g[x[0] + "s"].cpu()[page, place].to(F64)
                big = w.abs().amax(-1)
                assert ((s - big / 127).abs() <= (2 * eps if x == "kp" else 2.0 ** -20) * big / 127).all()
                assert not ((y.to(F64) * s[:, None] - w).abs() > 0.5 * s[:, None] * (1 + 2.0 ** -10) + 3 * eps * big[:, None]).any()
            was[page, place] = y
        assert torch.equal(got, was)                          # nothing else is written


ROPES = [dict(HQ=4, HK=2, D=128), dict(HQ=16, HK=2, D=256, rot=64), dict(HQ=3, HK=3, D=64), dict(HQ=5, HK=1, D=64, rot=16),
         dict(HQ=40, HK=8, D=128, rot=32), dict(HQ=2, HK=1, D=256, rot=0), dict(HQ=6, HK=2, D=256), dict(HQ=20, HK=4, D=64, rot=48)]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kw", ROPES, ids=str)
def test_rope_norm(kw, interleaved, int8):
    d = R.inputs(3, [5, 1, 0, 33, 2], [5, 100, 7, 50, 2], page=48, int8=int8, extra=3, **kw)
    check_rope(d, interleaved=interleaved)


@pytest.mark.parametrize("wtype", [BF16, torch.float32])
@pytest.mark.parametrize("freq", [torch.float32, F64])
def test_rope_norm_types_and_far_positions(wtype, freq):
    d = R.inputs(4, [3, 2], [3, 40], 4, 2, 128, wtype=wtype, freq=freq, theta=1e6)
    d["qw"], d["kw"] = d["qw"] - 1, d["kw"] - 1
    check_rope(d, offset=1.0, eps=1e-5)
    # positions next to 2^31: the fraction of a turn is right to 2^-21 of one, 3e-6 radians
    d = R.inputs(5, [3], [3], 4, 2, 128, wtype=wtype, freq=freq, theta=1e6, page=512)
    last = 2 ** 31 - 512 - 1
    d["lens"], d["table"] = torch.tensor([last], dtype=torch.int32), torch.ones(1, (last + 511) // 512, dtype=torch.int32)
    check_rope(d)


def test_rope_norm_one_token_and_many():
    check_rope(R.inputs(6, [1], [9000], 16, 2, 256, rot=64))
    check_rope(R.inputs(7, [700, 1, 300], [700, 3, 900], 16, 2, 256, rot=64, page=64))       # three of a workgroup's vectors a lane
    check_rope(R.inputs(8, [1500, 20], [1501, 20], 12, 2, 128))                               # two


@pytest.mark.parametrize("kw", [dict(HQ=16, HK=2, D=256, rot=64), dict(HQ=5, HK=1, D=64, rot=16), dict(HQ=6, HK=3, D=128), dict(HQ=1, HK=1, D=256, rot=0)])
@pytest.mark.parametrize("interleaved,int8", [(False, False), (True, False), (False, True), (True, True)])
def test_rope_norm_more_tokens_than_workgroups_are_held(kw, interleaved, int8):
    """Several tokens a workgroup: sequences that begin and end inside one, no place, bad pages, rows of no sequence at the end."""
    d = R.inputs(13, [1500, 1, 2, 999, 5], [1500, 7, 0, 1203, 3], page=32, int8=int8, extra=3, **kw)
    d["table"][0, 3], d["table"][3, 20], d["table"][3, 21] = -1, d["kp"].shape[0], 2 ** 31 - 1
    check_rope(d, interleaved=interleaved, offset=0.5)


@pytest.mark.parametrize("kw", [dict(HQ=16, HK=2, D=256, rot=64), dict(HQ=5, HK=1, D=64, rot=16), dict(HQ=6, HK=3, D=128), dict(HQ=1, HK=1, D=256, rot=0)])
@pytest.mark.parametrize("interleaved,int8", [(False, False), (True, False), (False, True), (True, True)])
def test_rope_norm_more_tokens_than_workgroups_are_held(kw, interleaved, int8):
    """Several tokens a workgroup: sequences that begin and end inside one, no place, bad pages, rows of no sequence at the end."""
    d = R.inputs(13, [1500, 1, 2, 999, 5], [1500, 7, 0, 1203, 3], page=32, int8=int8, extra=3, **kw)
    d["table"][0, 3], d["table"][3, 20], d["table"][3, 21] = -1, d["kp"].shape[0], 2 ** 31 - 1
    check_rope(d, interleaved=interleaved, offset=0.5)


def test_rope_norm_padding_and_bad_pages():
    d = R.inputs(9, [4, 3, 6], [0, 2, 40], 4, 2, 128, extra=2)          # no place at all; two of three tokens; all
    check_rope(d)
    d = R.inputs(10, [40, 20], [40, 20], 4, 2, 128)
    d["table"][0, 1], d["table"][1, 0] = -1, d["kp"].shape[0]
    check_rope(d)
    d["table"][1, 1] = 2 ** 31 - 1
    d["loc"] = torch.tensor([-5, 35, 1000], dtype=torch.int32)           # held to the packed tokens
    check_rope(d)


def test_rope_norm_strides_and_in_place():
    """Column ranges of a projection's output, q beside its gate, pages by head, out = q."""
    d = R.inputs(11, [9, 30], [9, 64], 4, 2, 128, page=32)
    T = d["q"].shape[0]
    g = R.cuda(d)
    wide = torch.zeros(T, 4 * 256 + 2 * 256 + 8, device="cuda", dtype=BF16)
    q = wide[:, :1024].view(T, 4, 256)[..., :128]
    k, v = wide[:, 1024:1280].view(T, 2, 128), wide[:, 1280:1536].view(T, 2, 128)
    for x, t in (("q", q), ("k", k), ("v", v)):
        t.copy_(g[x])
        g[x] = t
    for x in ("kp", "vp"):
        g[x] = g[x].transpose(1, 2).contiguous().transpose(1, 2)
    g["out"] = q
    wide[:, 128:256] = 3
    check_rope(d, g)
    assert (wide[:, 128:256] == 3).all()


def test_rope_norm_zero_heads_in_8_bits():
    d = R.inputs(12, [4], [4], 2, 2, 64, int8=True)
    d["k"][1], d["v"][1], d["v"][2, 0, 3] = 0, 0, INF
    g = R.cuda(d)
    rope(g)
    where = {t: (p, o) for t, p, o in R.rope(d)[2]}
    assert (g["kp"][where[1]] == 0).all() and (g["ks"][where[1]] == 0).all() and (g["vs"][where[1]] == 0).all()
    assert (g["vp"][where[2]][0] == 0).all() and torch.isinf(g["vs"][where[2]][0]) and torch.isfinite(g["vs"][where[2]][1])


# ---- attend ------------------------------------------------------------------------------------------------------------------
SHAPES = [(4, 2, 128), (16, 2, 256), (3, 3, 64), (5, 1, 64), (40, 8, 128), (6, 2, 256), (32, 1, 128), (40, 1, 64), (7, 1, 256)]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("HQ,HK,D", SHAPES)
def test_attend(HQ, HK, D, int8):
    """Single tokens, drafts, prompts from nothing and pieces of them in one batch; a sequence of none."""
    d = R.inputs(20, [1, 3, 0, 77, 1, 40, 9], [1, 90, 5, 77, 300, 171, 9], HQ, HK, D, page=48, int8=int8, extra=2, gate=HQ == 16)
    out = check_attend(d)
    assert (out.cpu()[-2:] == 7).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 33, 64, 100, 4096])
def test_attend_window(window, int8):
    check_attend(R.inputs(21, [1, 130, 4, 1], [200, 190, 70, 1], 8, 2, 128, page=16, int8=int8), window=window)
    check_attend(R.inputs(22, [1, 70, 4], [200, 190, 70], 4, 4, 64, page=32, int8=int8), window=window)
    check_attend(R.inputs(23, [2, 70], [90, 150], 4, 2, 256, page=32, int8=int8), window=window)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ctx", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257])
def test_attend_lengths_around_tiles(ctx, D):
    check_attend(R.inputs(24, [1, ctx], [ctx, ctx], 4, 2, D), longest=ctx)
    check_attend(R.inputs(25, [1], [ctx], 4, 2, D))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_long_contexts_in_pieces(D, int8):
    """Few rows over long contexts: the keys are split and joined, unevenly where sequences are short."""
    check_attend(R.inputs(26, [1], [5003], 8, 2, D, int8=int8), longest=1)
    check_attend(R.inputs(27, [1, 1, 2], [4100, 17, 2222], 4, 1, D, page=64, int8=int8, gate=True))
    check_attend(R.inputs(28, [50], [6000], 8, 2, D, int8=int8, gate=True))         # many rows, still fewer than the GPU has places
    check_attend(R.inputs(29, [1], [5003], 8, 2, D, int8=int8), longest=1, window=3000)


def test_attend_many_rows():
    """More row tiles than pieces are made for; all heads of a cache on one XCD, or not."""
    check_attend(R.inputs(30, [600, 3, 401], [600, 100, 700], 32, 4, 64, page=64))
    check_attend(R.inputs(31, [500], [520], 24, 8, 128, page=64))
    check_attend(R.inputs(32, [300, 200], [300, 300], 12, 3, 256, page=64))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("new", [[1, 1], [3, 2], [90, 70], [1, 90]], ids=str)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_is_not_seen_does_not_reach(new, D, int8):
    """NaN and infinities in keys and values behind a token, before its window and in the pages' unused places."""
    ctx = [n + 70 for n in new]
    d = R.inputs(33, new, ctx, 4, 2, D, page=48, int8=int8)
    clean = R.attend(d, window=50)
    hurt = dict(d)
    used = torch.zeros(d["kp"].shape[:2], dtype=torch.bool)
    for n, m in enumerate(ctx):
        page, place = R.page_rows(d, n, m - new[n] - 49, m)
        used[page, place] = True
    for x, bad in (("k", NAN), ("v", INF)):
        if int8:
            hurt[x + "s"] = torch.where(used[..., None], d[x + "s"], torch.full((), bad))
        else:
            hurt[x + "p"] = torch.where(used[..., None, None], d[x + "p"], torch.full((), bad, dtype=BF16))
    R.near(attend(R.cuda(hurt), window=50), *clean)
    # the last token's key and value: they reach its own rows alone
    clean = R.attend(d)
    for n, m in enumerate(ctx):
        (page,), (place,) = R.page_rows(d, n, m - 1, m)
        for x, bad in (("k", INF), ("v", NAN)):
            t = (hurt if n == 0 and x == "k" else hurt)
            if int8:
                t[x + "s"] = (d[x + "s"] if n == 0 else t[x + "s"]).clone()
                t[x + "s"][page, place] = NAN
                t[x + "p"] = d[x + "p"]
            else:
                t[x + "p"] = (d[x + "p"] if n == 0 else t[x + "p"]).clone()
                t[x + "p"][page, place] = bad
    out = attend(R.cuda(hurt)).cpu()
    last = [sum(new[:n + 1]) - 1 for n in range(len(new))]
    others = [t for t in range(sum(new)) if t not in last]
    assert torch.isnan(out[last]).all()
    if others:
        R.near(out[others], *(x[others] for x in clean))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_that_are_not_finite_reach_who_sees_them(D):
    """An infinite value in the middle of a prompt: rows from its token on, in its channel alone."""
    d = R.inputs(34, [80], [80], 4, 2, D)
    (page,), (place,) = R.page_rows(d, 0, 37, 38)
    want = R.attend(d)
    d["vp"][page, place, 1, 5] = -INF
    out = attend(R.cuda(d)).cpu()
    hit = torch.zeros(80, 4, D, dtype=torch.bool)
    hit[37:, 2:, 5] = True                                    # heads 2 and 3 read head 1
    assert (out[hit] == -INF).all()
    got = torch.where(hit, want[0].to(BF16), out)
    R.near(got, *want)


@pytest.mark.parametrize("new,ctx", [([6, 2], [3, 90]), ([70], [40]), ([90, 1], [60, 0])])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40])
def test_the_longest_windows_and_rows_before_the_first_position(new, ctx, window):
    check_attend(R.inputs(34, new, ctx, 4, 2, 128), window=window)


def test_attend_padding_and_rows_before_the_first_position():
    d = R.inputs(35, [2, 5, 3, 60], [0, 3, 0, 20], 8, 2, 128, extra=1)
    out = check_attend(d).cpu()
    assert (out[:2] == 0).all() and (out[2:4] == 0).all() and (out[7:10] == 0).all() and (out[10:50] == 0).all() and (out[-1] == 7).all()


def test_attend_offsets_are_held():
    d = R.inputs(36, [20, 30], [40, 60], 4, 2, 128)
    d["loc"] = torch.tensor([-7, 20, 10 ** 6], dtype=torch.int32)
    d["lens"] = torch.tensor([40, 10 ** 9], dtype=torch.int32)           # all that the table has
    check_attend(d)
    d["loc"] = torch.tensor([30, 10, 50], dtype=torch.int32)             # a sequence that would end before it begins
    d["lens"] = torch.tensor([40, -3], dtype=torch.int32)
    check_attend(d)


def test_attend_bad_pages_read_page_0():
    d = R.inputs(37, [1, 40], [90, 90], 4, 2, 128)
    d["table"][0, 2], d["table"][1, 3], d["table"][1, 5] = -1, d["kp"].shape[0], 2 ** 31 - 1
    check_attend(d)


@pytest.mark.parametrize("longest", [None, 1, 3, 90, 10 ** 6])
def test_longest_decides_on_speed_only(longest):
    d = R.inputs(38, [1, 90, 3], [700, 190, 64], 8, 2, 128)
    check_attend(d, longest=longest)
    check_attend(R.inputs(39, [90], [700], 8, 2, 64), longest=longest)


def test_attend_strides_and_in_place():
    d = R.inputs(40, [1, 50], [90, 80], 4, 2, 128, page=32, gate=True)
    want = R.attend(d)
    g = R.cuda(d)
    T = d["q"].shape[0]
    wide = torch.zeros(T, 4, 256, device="cuda", dtype=BF16)
    wide[..., :128], wide[..., 128:] = g["q"], g["gate"]
    g["q"], g["gate"] = wide[..., :128], wide[..., 128:]
    both = torch.stack([g["kp"], g["vp"]], 1).transpose(2, 3).contiguous()           # [pages, 2, heads, page, D]
    g["kp"], g["vp"] = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    g["out"] = g["q"]
    R.near(attend(g), *want)
    assert torch.equal(g["gate"].cpu(), d["gate"])
    # heads before tokens
    g = R.cuda(d)
    g["q"], g["out"] = (g[x].transpose(0, 1).contiguous().transpose(0, 1) for x in ("q", "out"))
    R.near(attend(g), *want)


def test_attend_index_types():
    d = R.inputs(41, [1, 20], [90, 80], 4, 2, 128)
    g = R.cuda(d)
    g["table"] = torch.cat([g["table"].long(), g["table"].long()], 1)[:, :d["table"].shape[1]]
    g["loc"], g["lens"] = g["loc"].long(), g["lens"].short()
    R.near(attend(g), *R.attend(d))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_scores_of_large_magnitude(D):
    """A maximum that grows along the keys, and weights that vanish: nothing overflows."""
    d = R.inputs(42, [1, 50], [500, 400], 4, 2, D)
    for n, m in enumerate((500, 400)):
        page, place = R.page_rows(d, n, 0, m)
        d["kp"][page, place] = (0.02 * torch.arange(m)[:, None, None] * d["kp"][page, place].float()).to(BF16)
    out = attend(R.cuda(d), scale=1.0)
    want, A, S = R.attend(d, scale=1.0)
    # scores of up to 400 by fp32 sums of D products: off by up to 2^-24 D^1/2 400 in the mean, a few times that at most
    assert torch.isfinite(out).all()
    err = (out.cpu().to(F64) - want).abs()
    assert not (err > 2.0 ** -8 * (want.abs() + A) + 2.0 ** -8 * A).any()
    # the largest score alone counts.  |q|, |k| < 5e15, 4e16: scores below 256 x 2e32 = 6e34, within fp32 (1e18 each would pass it)
    d["q"] = d["q"] * 1e15
    d["kp"] = d["kp"] * 1e15
    out = attend(R.cuda(d))
    assert torch.isfinite(out).all()


def test_attend_past_32_bit_offsets():
    """A cache of more than 2^31 elements, 4 GiB of keys: its last pages."""
    NP, page, HK, D = 70000, 16, 8, 256
    d = R.inputs(43, [1, 40], [90, 80], 16, 8, 256)
    g = R.cuda(d)
    few = d["kp"].shape[0]
    for x in ("kp", "vp"):
        big = torch.zeros(NP, page, HK, D, device="cuda", dtype=BF16)
        big[NP - few:] = g[x]
        g[x] = big
    g["table"] = g["table"] + NP - few
    R.near(attend(g), *R.attend(d))
    rope(g)
    _, k, where = R.rope(d)
    for t, p, o in where:
        assert torch.equal(g["vp"][NP - few + p, o].cpu(), d["v"][t])


def test_attend_on_a_side_stream_and_twice_at_once():
    """Two calls in flight on two streams, each with a workspace of its own."""
    ds = [R.inputs(44 + i, [1, 60], [3000 + 11 * i, 90], 8, 2, 128) for i in range(2)]
    gs = [R.cuda(d) for d in ds]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(gs, streams):
            with torch.cuda.stream(s):
                attend(g)
    torch.cuda.synchronize()
    for d, g in zip(ds, gs):
        R.near(g["out"], *R.attend(d))


def test_captured_calls():
    """rope_norm and attend in one graph, replayed as the batch moves on: lens and tables are read at the replay."""
    from leapquant_amd import attn
    d = R.inputs(50, [1, 1, 2], [2000, 40, 70], 8, 2, 128, page=16)
    d["table"] = torch.cat([d["table"], torch.zeros(3, 1, dtype=torch.int32)], 1)
    g = R.cuda(d)
    x, o = torch.empty_like(g["q"]), torch.empty_like(g["q"])

    def step():
        attn.rope_norm(g["q"], g["k"], g["v"], g["qw"], g["kw"], g["inv_freq"], pages(g), g["table"], g["loc"], g["lens"], x)
        attn.attend(x, pages(g), g["table"], g["loc"], g["lens"], o, longest=2)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    gen = torch.Generator().manual_seed(3)
    for i in range(5):
        for name in ("q", "k", "v"):
            g[name].copy_(torch.randn(d[name].shape, generator=gen).to(BF16))
        if i:
            g["lens"] += torch.tensor([1, 1, 2], device="cuda", dtype=torch.int32)
        o.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        now = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in g.items()}
        now["q"] = x.cpu()
        R.near(o, *R.attend(now))
        eager = o.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(eager, o)


def test_same_call_same_bits():
    d = R.inputs(51, [1, 90, 3], [3000, 190, 64], 8, 2, 128)
    a, b = attend(R.cuda(d)).clone(), attend(R.cuda(d))
    assert torch.equal(a, b)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("HQ,HK,D", [(16, 2, 256), (6, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("new,ctx", [([50], [6000]), ([200], [300]), ([3, 1, 77], [2000, 900, 77]), ([1, 1], [4099, 40])])
def test_calls_again_are_the_same_bits(new, ctx, HQ, HK, D, int8):
    """Row tiles that are not full, pieces of the keys and both kinds of sequences: four calls of the same inputs."""
    g = R.cuda(R.inputs(54, new, ctx, HQ, HK, D, int8=int8))
    outs = [attend(g).clone() for _ in range(4)]
    assert all(torch.equal(outs[0], x) for x in outs[1:])


@pytest.mark.parametrize("longest", [None, 90])
@pytest.mark.parametrize("new", [[90] + 20 * [1], [90, 40, 30, 1, 60], [1, 90, 16, 17, 3, 1]])
@pytest.mark.parametrize("HQ,HK,D,int8", [(16, 2, 256, False), (8, 2, 128, True), (8, 8, 64, False)])
def test_sequences_of_one_token_beside_longer_ones(new, longest, HQ, HK, D, int8):
    """With the longest's tokens said, the others' mean settles whether those of few rows have workgroups of their own."""
    ctx = [max(m, (37 * i * i) % 700) for i, m in enumerate(new)]
    check_attend(R.inputs(55, new, ctx, HQ, HK, D, int8=int8), longest=longest)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("factor", [1e-25, 1e-17, 1e17, 1e20])
def test_scales_of_any_size(factor, new, D):
    """Scales next to and beyond those whose inverse is taken, some of them zero, beside ordinary ones.  A weight's product
    with its scale and codes stays within fp32 throughout (1e20 127 2^8)."""
    d = R.inputs(56, [new], [200], 4, 2, D, int8=True)
    d["vs"][::2] *= factor
    d["vs"][1::4, 3] = 0
    check_attend(d)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("HQ,HK,D", [(16, 2, 256), (6, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("new,ctx", [([50], [6000]), ([200], [300]), ([3, 1, 77], [2000, 900, 77]), ([1, 1], [4099, 40])])
def test_calls_again_are_the_same_bits(new, ctx, HQ, HK, D, int8):
    """Row tiles that are not full, pieces of the keys and both kinds of sequences: four calls of the same inputs."""
    g = R.cuda(R.inputs(54, new, ctx, HQ, HK, D, int8=int8))
    outs = [attend(g).clone() for _ in range(4)]
    assert all(torch.equal(outs[0], x) for x in outs[1:])


@pytest.mark.parametrize("longest", [None, 90])
@pytest.mark.parametrize("new", [[90] + 20 * [1], [90, 40, 30, 1, 60], [1, 90, 16, 17, 3, 1]])
@pytest.mark.parametrize("HQ,HK,D,int8", [(16, 2, 256, False), (8, 2, 128, True), (8, 8, 64, False)])
def test_sequences_of_one_token_beside_longer_ones(new, longest, HQ, HK, D, int8):
    """With the longest's tokens said, the others' mean settles whether those of few rows have workgroups of their own."""
    ctx = [max(m, (37 * i * i) % 700) for i, m in enumerate(new)]
    check_attend(R.inputs(55, new, ctx, HQ, HK, D, int8=int8), longest=longest)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("factor", [1e-25, 1e-17, 1e17, 1e20])
def test_scales_of_any_size(factor, new, D):
    """Scales next to and beyond those whose inverse is taken, some of them zero, beside ordinary ones.  A weight's product
    with its scale and codes stays within fp32 throughout (1e20 127 2^8)."""
    d = R.inputs(56, [new], [200], 4, 2, D, int8=True)
    d["vs"][::2] *= factor
    d["vs"][1::4, 3] = 0
    check_attend(d)


def test_empty_calls():
    d = R.inputs(52, [1], [5], 4, 2, 128)
    g = R.cuda(d)
    none = dict(g, q=g["q"][:0], k=g["k"][:0], v=g["v"][:0], out=g["out"][:0], loc=g["loc"] * 0)
    attend(none)
    rope(none)
    none = dict(g, table=g["table"][:0], loc=g["loc"][:1], lens=g["lens"][:0])
    attend(none)
    rope(none)
    torch.cuda.synchronize()
    assert (g["out"] == 7).all()


def test_sine_and_cosine():
    """The hardware's, of a fraction of a turn, through a head of ones: (cos - sin, cos + sin) at bf16, so by pages of steps."""
    d = R.inputs(53, [4096], [4096], 1, 1, 64, freq=F64, theta=3e3, page=64, wtype=torch.float32)
    check_rope(d)


# ---- together: a layer over prompts in pieces, then tokens ---------------------------------------------------------------------
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("window", [0, 60])
def test_a_layer_in_pieces_is_the_layer(window, int8):
    """Two sequences, their prompts in pieces and decode tokens beside each other, against the whole sequences at once in 64 bits."""
    from leapquant_amd import attn
    HQ, HK, D, page, lens = 8, 2, 128, 16, (150, 90)
    full = R.inputs(60, list(lens), list(lens), HQ, HK, D, page=page, int8=int8, gate=True)
    g = R.cuda(full)
    at = [0, 0]
    outs = [[], []]
    start = [0, lens[0]]
    first_pieces = [(64, 30), (64, 1), (1, 1), (1, 40), (3, 1), (1, 1), (16, 16)]
    for new in first_pieces:
        rows = torch.cat([torch.arange(start[n] + at[n], start[n] + at[n] + new[n]) for n in range(2)]).cuda()
        at = [a + m for a, m in zip(at, new)]
        assert at[0] <= lens[0] and at[1] <= lens[1]
        loc = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device="cuda")
        now = torch.tensor(at, dtype=torch.int32, device="cuda")
        x = torch.empty(sum(new), HQ, D, device="cuda", dtype=BF16)
        attn.rope_norm(g["q"][rows], g["k"][rows], g["v"][rows], g["qw"], g["kw"], g["inv_freq"], pages(g), g["table"], loc, now, x)
        attn.attend(x, pages(g), g["table"], loc, now, x, window=window, gate=g["gate"][rows], longest=max(new))
        outs[0].append(x[:new[0]])
        outs[1].append(x[new[0]:])
    assert at == [150, 90]
    got = torch.cat(outs[0] + outs[1]).cpu()
    # the layer's definition: keys and queries not rounded in between.  A score of |q| |k| D^-1/2 = D^1/2 moves by 2 x 2^-8 of it in the
    # worst case and about 2^-8 in the mean (two roundings of random sign over D channels: 2^-8 / 3^1/2 each); codes of 8 bits move a key
    # and a value by 1/254 of its head's largest, here about 3.
    q, k, _ = R.rope(full)
    d = dict(full, q=q, ks=None, vs=None, kp=torch.zeros(full["kp"].shape, dtype=F64), vp=torch.zeros(full["kp"].shape, dtype=F64))
    for t, page, place in R.rope(full)[2]:
        d["kp"][page, place], d["vp"][page, place] = k[t], full["v"][t].to(F64)
    want, A, S = R.attend(d, window=window)
    err = (got.to(F64) - want).abs()
    step = 1.5 / 127 if int8 else 0.0
    assert float(err.norm()) <= (2.0 ** -6 + 2 * step) * float((want * want + S * S).sum().sqrt())
    # and against what the cache holds, by the operators' own bars
    now = {n: v.cpu() if isinstance(v, torch.Tensor) else v for n, v in g.items()}
    now["q"] = R.rope(full)[0].to(BF16)
    R.near(got[-40:], *(x[-40:] for x in R.attend(now, window=window)))


# ---- the start of a walk over tiles of keys ------------------------------------------------------------------------------------
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("HQ,HK,D", [(16, 2, 256), (8, 2, 128), (4, 4, 64)])
def test_warm_calls_of_part_full_tiles(HQ, HK, D, int8):
    """Waves without rows beside waves with rows, walks of three tiles of keys and more: the first call is right, and calls whose
    keys lie in the L2 are the same bits.  (Which write comes before which read in LDS: tests/test_attn_order.py.)"""
    G = HQ // HK
    for new, ctx in (([20 // G + 17], [400]), ([33 + 128 // G, 40], [500, 130]), ([100], [100 + 64 * 3])):
        d = R.inputs(57, new, ctx, HQ, HK, D, int8=int8, page=32)
        g = R.cuda(d)
        first = attend(g, longest=max(new)).clone()
        R.near(first, *R.attend(d))
        same = torch.stack([(attend(g, longest=max(new)) == first).all() for _ in range(30)])
        assert same.all()


# ---- 8-bit pages hide nothing ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [[6, 40], [2030, 90]], ids=["few", "many"])          # a token a workgroup, and several
def test_nan_goes_through_8_bit_pages(new, D, interleaved):
    """A NaN in a head of a key or value makes that head's scale NaN and its codes 0, an infinity beside it or not; the tokens
    that see it have NaN in the query heads that read it, all others what they had."""
    d = R.inputs(58, new, new, 4, 2, D, page=32, int8=True)
    T, last = sum(new), new[0] - 2
    d["k"][last, 1, D - 3] = NAN                     # a key's head is NaN as a whole after its norm
    d["v"][T - 5, 0, D // 2 + 1], d["v"][T - 5, 0, 7] = NAN, INF
    g = R.cuda(d)
    rope(g, interleaved=interleaved)
    clean = dict(d, k=torch.nan_to_num(d["k"], 0.0, 0.0), v=torch.nan_to_num(d["v"], 0.0, 0.0))
    _, k, where = R.rope(clean, interleaved=interleaved)
    got = {x: g[x].cpu() for x in ("kp", "vp", "ks", "vs")}
    for t, page, place in where:
        for x, vals, bad in (("k", k, (last, 1)), ("v", d["v"].to(F64), (T - 5, 0))):
            for h in range(2):
                s, c = got[x + "s"][page, place, h], got[x + "p"][page, place, h]
                if (t, h) == bad:
                    assert torch.isnan(s) and (c == 0).all(), (x, t, h)
                else:
                    big = float(vals[t, h].abs().amax())
                    # the head's largest by test_rope_norm's bar, 2^-16 of it, and the scale's own rounding
                    assert abs(float(s) - big / 127) <= 2.0 ** -15 * big / 127, (x, t, h)
    out = attend(g).cpu()
    hit = torch.zeros(T, 4, D, dtype=torch.bool)
    hit[last:new[0], 2:] = True
    hit[T - 5:, :2] = True
    assert torch.isnan(out[hit]).all() and torch.isfinite(out[~hit]).all()


def test_heads_of_next_to_nothing_in_8_bits():
    """Heads whose largest is at most 1e-30 have scales and codes of 0, the next larger ones have neither."""
    d = R.inputs(59, [6], [6], 2, 2, 64, int8=True)
    d["v"] *= 0
    tiny = torch.tensor([1e-30, 1e-38, 1.01e-30, 1e-29, -1e-30, -1.01e-30]).to(BF16)
    d["v"][:, :, 5] = tiny[:, None]
    g = R.cuda(d)
    rope(g)
    for t, page, place in R.rope(d)[2]:
        s, c = g["vs"][page, place].cpu(), g["vp"][page, place].cpu()
        big = abs(float(tiny[t]))
        if big <= 1e-30:
            assert (s == 0).all() and (c == 0).all(), t
        else:
            # one rounding of 1 / 127 and one of the product
            assert ((s.to(F64) - big / 127).abs() <= 2.0 ** -23 * big / 127).all() and (c[:, 5].abs() == 127).all(), t


# ---- outputs of rows before the first position ------------------------------------------------------------------------------
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,ctx", [([2, 5, 1], [0, 3, 40]), ([70, 60], [0, 20]), ([1, 90, 2], [3000, 60, 0]), ([3, 2], [1, 5000])])
def test_padding_is_zero_whatever_its_gate_holds(new, ctx, D, int8):
    """Sequences without cached tokens, and partly before position 0, whose queries and gates hold NaN and infinities: alone, beside others, and
    where keys are split and joined."""
    d = R.inputs(61, new, ctx, 8, 2, D, int8=int8, gate=True)
    none = torch.zeros(sum(new), dtype=torch.bool)
    for lo, m, all_ in R.batch(d):
        none[lo:lo + max(m - all_, 0)] = True
    want = R.attend(d)
    assert none.any() and (want[0][none] == 0).all()
    for bad in (NAN, INF, -INF):
        d["gate"][none] = d["q"][none] = bad
        for longest in (None, max(new)):
            out = attend(R.cuda(d), longest=longest)
            assert (out.cpu()[none] == 0).all(), bad
            R.near(out, *want)


# ---- indexes of other integer types ------------------------------------------------------------------------------------------
def test_wide_indexes_do_not_wrap():
    """int64 tables, offsets and lengths past 32 bits are held to what there is, as those within."""
    far = 2 ** 32
    d = R.inputs(62, [5, 40, 3], [30, 60, 20], 4, 2, 128)
    d["table"] = d["table"].long()
    d["table"][0, 1], d["table"][1, 3], d["table"][1, 0], d["table"][2, 1] = far + 1, -far + 1, -2 ** 63, 2 ** 63 - 1
    d["loc"] = torch.tensor([-far, 5, 45, far + 46])          # the last one to T
    d["lens"] = torch.tensor([30, far + 7, -far + 20])        # all that the table has; none
    check_attend(d)
    check_rope(d)
    small = R.inputs(63, [5, 3], [30, 20], 4, 2, 128)
    for t in (torch.uint8, torch.int16, torch.uint16, torch.uint32, torch.uint64):
        check_attend(dict(small, table=small["table"].to(t), loc=small["loc"].to(t), lens=small["lens"].to(t)))
    for t, n in ((torch.uint32, 2 ** 32 - 1), (torch.uint64, 2 ** 64 - 5)):
        d = R.inputs(63, [5, 3], [30, 20], 4, 2, 128)
        g = R.cuda(d)
        d["table"][0, 1], d["lens"][1], d["loc"][2] = -1, 10 ** 9, 10 ** 9
        for x, at in (("table", (0, 1)), ("lens", 1), ("loc", 2)):
            g[x] = g[x].to(t)
            g[x][at] = torch.tensor(n, dtype=t)
        R.near(attend(g), *R.attend(d))


def test_wide_indexes_in_a_graph():
    """A captured call converts the indexes at every replay."""
    d = R.inputs(64, [1, 40], [300, 60], 4, 2, 128)
    g = R.cuda(d)
    for x in ("table", "loc", "lens"):
        g[x] = g[x].long()
    attend(g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(g)
    for n in (300, 170, 2 ** 33):
        g["lens"][0] = n
        g["out"].fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        d["lens"][0] = min(n, 10 ** 9)
        R.near(g["out"], *R.attend(d))


# ---- layouts ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,ctx", [([1, 3], [400, 90]), ([70, 1], [200, 90])])
def test_layouts_of_pages_and_tables(new, ctx):
    """Codes and scales by head, scales beside each other in one tensor, a table that is a column range of a wider one."""
    d = R.inputs(65, new, ctx, 8, 2, 128, page=32, int8=True)
    NP, page, HK, D = d["kp"].shape
    g = R.cuda(d)
    codes = torch.stack([g["kp"], g["vp"]], 1).transpose(2, 3).contiguous()              # [pages, 2, heads, page, D]
    scales = torch.zeros(HK, NP, 2, page, 3, device="cuda")
    for i, x in enumerate(("k", "v")):
        g[x + "p"] = codes[:, i].transpose(1, 2)
        s = scales[:, :, i, :, 1].permute(1, 2, 0)                                        # head-major, three floats apart
        s.copy_(g[x + "s"])
        g[x + "s"] = s
    wide = torch.full((len(new), d["table"].shape[1] + 5), 2 ** 30, dtype=torch.int32, device="cuda")
    wide[:, 2:-3] = g["table"]
    g["table"] = wide[:, 2:-3]
    assert g["table"].stride(0) > g["table"].shape[1]
    for longest in (None, max(new)):
        R.near(attend(g, longest=longest), *R.attend(d))
    check_rope(d, g)
    assert (scales[..., 0] == 0).all() and (scales[..., 2] == 0).all()


def test_8_bit_pages_past_32_bit_offsets():
    """Codes of more than 2^32 bytes and scales beside them: the last pages."""
    NP, page, HK, D = 140000, 16, 8, 256
    d = R.inputs(66, [1, 40, 3], [90, 80, 3], 16, 8, 256, int8=True)
    g = R.cuda(d)
    few = d["kp"].shape[0]
    for x in ("kp", "vp", "ks", "vs"):
        big = torch.zeros((NP,) + tuple(d[x].shape[1:]), device="cuda", dtype=d[x].dtype)
        big[NP - few:] = g[x]
        g[x] = big
    assert g["kp"].numel() > 2 ** 32
    g["table"] = g["table"] + NP - few
    R.near(attend(g), *R.attend(d))
    rope(g)
    last = {x: g[x][NP - few:].cpu() for x in ("kp", "vp", "ks", "vs")}
    assert not any(g[x][:NP - few].any() for x in ("kp", "vp"))
    for t, p, o in R.rope(d)[2]:
        w = d["v"][t].to(F64)
        s = last["vs"][p, o].to(F64)[:, None]
        assert not ((last["vp"][p, o].to(F64) * s - w).abs() > 0.5 * s * (1 + 2.0 ** -10) + 2.0 ** -17 * w.abs().amax(-1, keepdim=True)).any()
    del g, big                                # what lasts of later tests would lie in these segments and keep them
    torch.cuda.empty_cache()


# ---- more sequences than a wave has lanes -------------------------------------------------------------------------------------
@pytest.mark.parametrize("N", [65, 150, 4200])
def test_many_sequences(N):
    """The search for a token's and a row tile's sequence takes two and three steps; empty sequences, padding, a few longer ones."""
    gen = torch.Generator().manual_seed(N)
    new = torch.randint(0, 3, (N,), generator=gen).tolist()
    ctx = [m + int(x) for m, x in zip(new, torch.randint(0, 20, (N,), generator=gen))]
    for n in (0, N // 2, N - 1):
        new[n], ctx[n] = 70, 90
    ctx[3] = ctx[N - 2] = 0
    for longest in (None, 70):
        check_attend(R.inputs(67, new, ctx, 2, 1, 64, extra=2), longest=longest)
    check_rope(R.inputs(68, new, ctx, 2, 1, 64, extra=2))
