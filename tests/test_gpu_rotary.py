"""qk_rotary on the GPU against its definition in 64 bits: norms, pairings, axes, text before and
after, heads of their own for k, layouts, in place, on other streams and in graphs."""

import pytest
import torch

import recap_amd
from around_util import check, qk
from recap_amd import kernels as K

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
CHANNELS = {64: (16, 24, 24), 128: (44, 42, 42)}


def make(seed, batch, heads, tokens, d, dtype=BF, norm=None, heads_k=None, wtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    out = {}
    for name, h in (("q", heads), ("k", heads if heads_k is None else heads_k)):
        size = (0.4 * rand(h, 1, d)).exp()
        out[name] = ((rand(batch, h, tokens, d) + 0.2) * size).to(dtype)
        if norm:
            extent = h * d if norm == "rms_all" else d
            out[f"{name}_weight"] = (1 + 0.3 * rand(extent)).to(wtype or dtype)
            out[f"{name}_bias"] = (0.3 * rand(extent)).to(wtype or dtype)
    return out


def run(a, axes, **more):
    named = {n: v for n, v in a.items() if n not in ("q", "k")}
    return K.qk_rotary(a["q"], a.get("k"), axes, **named, **more)


def check_both(a, axes, label, *, norm=None, offset=0, pairing="interleaved"):
    print(f"case {label} {norm} {pairing} offset {offset} {tuple(a['q'].shape)}", flush=True)
    got = run(a, axes, norm=norm, offset=offset, pairing=pairing)
    for name, out in zip(("q", "k"), got):
        want = qk(a[name], axes, offset=offset, pairing=pairing, kind=norm,
                  weight=a.get(f"{name}_weight"), bias=a.get(f"{name}_bias"))
        assert out.dtype == a[name].dtype and out.is_contiguous()
        check(out, want, f"{label} {name}")
    return got


@pytest.mark.parametrize("norm", [None, "rms", "layer", "rms_all"])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("d,dtype", [(64, BF), (64, FP), (128, BF), (128, FP)])
def test_norms_and_pairings(cuda, norm, pairing, d, dtype):
    axes = recap_amd.rotary_axes((3, 5, 7), CHANNELS[d], device=cuda)
    for offset, wtype in ((0, dtype), (13, F32)):
        a = make(1, 2, 3, 105 + 13 + 4, d, dtype, norm, wtype=wtype)
        check_both(a, axes, f"{dtype}", norm=norm, offset=offset, pairing=pairing)


@pytest.mark.parametrize("grid,channels", [
    ((1, 1, 1), (44, 42, 42)), ((1, 9, 4), (0, 64, 64)), ((7, 1, 1), (128, 0, 0)),
    ((2, 3, 4), (2, 124, 2)), ((1, 1, 300), (0, 0, 128)), ((33, 2, 5), (16, 56, 56)),
    ((4, 11, 3), (126, 0, 2))])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
def test_axes(cuda, grid, channels, pairing):
    axes = recap_amd.rotary_axes(grid, channels, positions=[None, None, [0.37 * i for i in
                                                                       range(grid[2])]],
                                 device=cuda)
    n = grid[0] * grid[1] * grid[2]
    check_both(make(2, 1, 2, n, 128, norm="rms"), axes, f"{grid} {channels}", norm="rms",
               pairing=pairing)
    check_both(make(3, 2, 1, n + 5, 128), axes, f"{grid} {channels}", offset=5, pairing=pairing)


@pytest.mark.parametrize("batch,heads,tokens", [(1, 1, 1), (1, 1, 2), (3, 2, 1), (1, 48, 17), (2, 5, 129),
                                                (1, 24, 1025), (1, 12, 3001), (1, 130, 9)])
@pytest.mark.parametrize("norm", ["rms", "rms_all"])
@pytest.mark.parametrize("d", [64, 128])
def test_sizes(cuda, batch, heads, tokens, norm, d):
    """Without axes the tokens are only normalised; with a grid of all of them, all turn."""
    a = make(4, batch, heads, tokens, d, norm=norm)
    check_both(a, None, "no axes", norm=norm)
    check_both(a, recap_amd.rotary_axes((1, 1, tokens), CHANNELS[d], device=cuda), "one line",
               norm=norm)


@pytest.mark.parametrize("norm", [None, "layer", "rms_all"])
def test_heads_of_their_own(cuda, norm):
    """k with fewer or more heads than q, and q alone."""
    axes = recap_amd.rotary_axes((2, 4, 5), CHANNELS[64], device=cuda)
    for heads_k in (1, 3, 20):
        a = make(5, 2, 8, 44, 64, norm=norm, heads_k=heads_k)
        got = check_both(a, axes, f"k heads {heads_k}", norm=norm, offset=2)
        alone, none = run({n: v for n, v in a.items() if n[0] == "q"}, axes, norm=norm, offset=2)
        assert none is None and torch.equal(alone, got[0])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("norm", [None, "rms", "rms_all"])
def test_layouts(cuda, d, norm):
    """Views of projections, fused projections, expanded and misaligned inputs, outputs in place
    and as parts of a longer sequence: all equal the contiguous call bit for bit."""
    axes = recap_amd.rotary_axes((2, 4, 5), CHANNELS[d], device=cuda)
    b, h, n, off = 2, 3, 47, 7
    a = make(6, b, h, n, d, norm=norm)
    rest = {key: v for key, v in a.items() if len(key) > 1}
    want = run(a, axes, norm=norm, offset=off)
    flat = {m: a[m].transpose(1, 2).reshape(b, n, h * d) for m in "qk"}
    fused = torch.stack([a["q"].transpose(1, 2), a["k"].transpose(1, 2), torch.ones_like(
        a["q"].transpose(1, 2))], dim=2)
    odd = torch.zeros(b, n, h * d + 1, dtype=BF, device=cuda)
    layouts = {"projection": {m: flat[m].view(b, n, h, d).transpose(1, 2) for m in "qk"},
               "fused": {m: fused[:, :, i].transpose(1, 2) for i, m in enumerate("qk")}}
    for label, tensors in layouts.items():
        print(f"case {label}", flush=True)
        got = run({**tensors, **rest}, axes, norm=norm, offset=off)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), label
        assert all(x.transpose(1, 2).is_contiguous() for x in got), label
        run({**tensors, **rest}, axes, norm=norm, offset=off, q_out=tensors["q"], k_out=tensors["k"])
        assert all(torch.equal(tensors[m], y) for m, y in zip("qk", want)), label
    assert torch.equal(fused[:, :, 2], torch.ones_like(fused[:, :, 2]))
    odd[:, :, 1:] = a["q"].transpose(1, 2).reshape(b, n, h * d)
    view = odd[:, :, 1:].unflatten(2, (h, d)).transpose(1, 2)
    assert torch.equal(run({**a, "q": view}, axes, norm=norm, offset=off)[0], want[0])
    apart = torch.zeros(2, h * n * d + 4, dtype=BF, device=cuda)   # an odd pitch of a batch of one
    apart[0, :h * n * d] = a["q"][0].reshape(-1)
    single = apart.as_strided((1, h, n, d), (apart.stride(0), n * d, d, 1))
    assert single.stride(0) % 8 == 4
    assert torch.equal(run({"q": single, **{m: v for m, v in rest.items() if m[0] == "q"}}, axes, norm=norm,
                           offset=off)[0][0], want[0][0])
    one = run({**a, "q": a["q"][:1].expand(b, h, n, d)}, axes, norm=norm, offset=off)[0]
    assert torch.equal(one[1], want[0][0])
    whole = torch.full((b, h, n + 9, d), 5.0, dtype=BF, device=cuda)
    run(a, axes, norm=norm, offset=off, q_out=whole[:, :, 4:4 + n])
    assert torch.equal(whole[:, :, 4:4 + n], want[0])
    assert (whole[:, :, :4] == 5).all() and (whole[:, :, 4 + n:] == 5).all()
    with pytest.raises(ValueError, match="overlaps"):
        run(a, axes, norm=norm, offset=off, q_out=a["k"])
    with pytest.raises(ValueError, match="aligned"):
        run(a, axes, norm=norm, offset=off, q_out=view)


@pytest.mark.parametrize("norm", [None, "rms_all"])
@pytest.mark.parametrize("dim", [0, 1, 2])
def test_expanded_inputs(cuda, dim, norm):
    """q and k with one batch, head or token expanded to all (a stride of 0) are read in place,
    also where another argument needs a copy."""
    a = make(16, 2, 3, 47, 64, norm=norm)
    axes = recap_amd.rotary_axes((2, 4, 5), CHANNELS[64], device=cuda)
    whole = {m: v.narrow(dim, 0, 1).expand_as(v) if len(m) == 1 else v for m, v in a.items()}
    assert whole["q"].stride(dim) == 0
    want = run({m: v.contiguous() for m, v in whole.items()}, axes, norm=norm, offset=5)
    got = run(whole, axes, norm=norm, offset=5)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    apart = [torch.stack((t, t), -1)[..., 0] for t in axes]
    got = run(whole, apart, norm=norm, offset=5)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_empty_and_refused(cuda):
    x = torch.zeros(0, 2, 5, 64, dtype=BF, device=cuda)
    assert K.qk_rotary(x, x)[1].shape == x.shape
    x = torch.zeros(1, 2, 5, 64, dtype=BF, device=cuda)
    with pytest.raises(ValueError, match="heads"):
        K.qk_rotary(x, x[:, :0])
    with pytest.raises(ValueError, match="GPU"):
        K.qk_rotary(x, x, recap_amd.rotary_axes((1, 1, 5), CHANNELS[64]))
    with pytest.raises(ValueError, match="gradient"):
        K.qk_rotary(x.clone().requires_grad_())
    with torch.no_grad():
        K.qk_rotary(x.clone().requires_grad_())


def test_values_that_are_not_numbers(cuda):
    """Infinities and NaN reach their own head's row (the token's, with a norm over all heads)."""
    for norm in (None, "rms", "layer", "rms_all"):
        a = make(7, 1, 2, 6, 64, norm=norm)
        axes = recap_amd.rotary_axes((1, 2, 3), CHANNELS[64], device=cuda)
        clean = run(a, axes, norm=norm)[0]
        a["q"][0, 0, 2, 5] = float("nan")
        a["q"][0, 1, 4, 9] = float("inf")
        got = run(a, axes, norm=norm)[0]
        hit = torch.zeros(2, 6, dtype=torch.bool, device=cuda)
        hit[0, 2] = hit[1, 4] = True
        if norm == "rms_all":
            hit[:, 2] = hit[:, 4] = True
        assert torch.equal(got[0][~hit], clean[0][~hit]), norm
        assert torch.isnan(got[0, 0, 2]).any() and not torch.isfinite(got[0, 1, 4]).all()


@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("d", [64, 128])
def test_tokens_outside_the_grid_keep_their_values(cuda, d, pairing):
    """Text tokens without a norm come out bit for bit, whatever stands beside a value: an
    infinity and a NaN stay in their own channel; a call without axes copies."""
    a = make(15, 2, 3, 40, d)
    q = a["q"]
    q[0, 1, 2, 8] = float("inf")
    q[1, 0, 3, 17] = float("nan")
    q[0, 2, 39, d - 1] = float("-inf")
    q[1, 2, 38, 0] = -0.0
    axes = recap_amd.rotary_axes((2, 3, 5), CHANNELS[d], device=cuda)
    got = K.qk_rotary(q, None, axes, offset=5, pairing=pairing)[0]
    for rows in (slice(0, 5), slice(35, 40)):
        assert torch.equal(got[:, :, rows].view(torch.int16), q[:, :, rows].view(torch.int16))
    assert torch.equal(K.qk_rotary(q, pairing=pairing)[0].view(torch.int16), q.view(torch.int16))


@pytest.mark.parametrize("norm", ["rms", "rms_all"])
@pytest.mark.parametrize("heads", [1, 12, 65, 4099])
def test_large_values(cuda, heads, norm):
    """Values just inside 1e17, at their signs' random turns: a norm over all heads adds heads * d
    squares, past fp32's range from some 270 heads of 128 on if they are added as they are."""
    g = torch.Generator(device="cuda").manual_seed(17)
    q = torch.randint(0, 2, (1, heads, 5, 128), generator=g, device="cuda").mul(2).sub(1).to(BF) * 9.9e16
    q = torch.cat((q, q / 3), dim=2)
    axes = recap_amd.rotary_axes((1, 2, 3), CHANNELS[128], device=cuda)
    check_both({"q": q, "k": q.flip(1)}, axes, f"{heads} heads", norm=norm, offset=2)


def test_streams_and_graph(cuda):
    axes = recap_amd.rotary_axes((3, 20, 20), CHANNELS[128], device=cuda)
    a = make(8, 1, 6, 1250, 128, norm="rms_all")
    fresh = [make(9 + i, 1, 6, 1250, 128, norm="rms_all") for i in range(3)]
    call = lambda x: run(x, axes, norm="rms_all", offset=50)  # noqa: E731
    want = call(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(a)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(a)
    for f in fresh:
        want = call(f)
        torch.cuda.synchronize()
        for n, v in f.items():
            a[n].copy_(v)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_offsets_beyond_32_bits(cuda):
    """Elements past 2^32: the last head and rows equal the same rows alone."""
    n, h, d = 1_500_000, 24, 128
    q = torch.zeros(1, h, n, d, dtype=BF, device=cuda)
    assert q.numel() > 2 ** 32
    tail = make(12, 1, h, 11, d, norm="rms")
    q[:, :, -11:] = tail["q"]
    axes = recap_amd.rotary_axes((1, 1, 11), CHANNELS[d], device=cuda)
    weight = tail["q_weight"]
    want = K.qk_rotary(tail["q"], None, axes, norm="rms", q_weight=weight)[0]
    got = K.qk_rotary(q, None, axes, offset=n - 11, norm="rms", q_weight=weight, q_out=q)[0]
    assert torch.equal(got[:, :, -11:], want) and not got[:, :, :-11].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("norm", [None, "rms", "layer", "rms_all"])
def test_large_calls_equal_small_ones(cuda, d, norm):
    """A call large enough to pass the caches by gives each token what a call of its own does."""
    h, n = 12, 3 * 64 * 100 * 128 // d
    a = make(13, 1, h, n, d, norm=norm)
    axes = recap_amd.rotary_axes((3, 1, n // 3), CHANNELS[d], device=cuda)
    whole = run(a, axes, norm=norm)
    for first in (0, n // 3 - 5, n - 9):
        where = [torch.arange(first, first + 9) // (n // 3), torch.arange(first, first + 9) % (n // 3)]
        rows = slice(first, first + 9)
        for i in range(9):   # a grid of one position, the token's own
            one = (axes[0][where[0][i]][None], axes[1], axes[2][where[1][i]][None])
            part = {m: v[:, :, first + i:first + i + 1] if len(m) == 1 else v for m, v in a.items()}
            got = run(part, one, norm=norm)
            assert all(torch.equal(x, y[:, :, rows][:, :, i:i + 1]) for x, y in zip(got, whole))


def test_more_tokens_than_one_launch(cuda):
    """Tokens beyond a launch's 2^20 workgroups (of 4 tokens each with 16 heads of 64)."""
    n = (1 << 22) + 50
    q = torch.zeros(1, n, 16, 64, dtype=BF, device=cuda).transpose(1, 2)
    tail = make(14, 1, 16, 40, 64, norm="rms")
    q[:, :, -40:] = tail["q"]
    axes = recap_amd.rotary_axes((1, 2, 20), CHANNELS[64], device=cuda)
    want = K.qk_rotary(tail["q"], None, axes, norm="rms", q_weight=tail["q_weight"])[0]
    got = K.qk_rotary(q, None, axes, offset=n - 40, norm="rms", q_weight=tail["q_weight"], q_out=q)[0]
    assert torch.equal(got[:, :, -40:], want) and not got[:, :, :-40].any()


@pytest.mark.parametrize("d,heads,heads_k,tokens", [
    (128, 48, 48, 70), (128, 48, 7, 70), (64, 130, 48, 33), (128, 41, 41, 70), (64, 80, 3, 1)])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
def test_many_heads_under_one_norm(cuda, d, heads, heads_k, tokens, pairing):
    """A norm over more heads than a wave holds at once reads them again after the sum: against the
    definition, and in place."""
    axes = recap_amd.rotary_axes((1, 1, tokens), CHANNELS[d], device=cuda)
    a = make(18, 2, heads, tokens, d, norm="rms_all", heads_k=heads_k)
    want = check_both(a, axes, f"{heads} and {heads_k} heads", norm="rms_all", pairing=pairing)
    b = {**a, "q": a["q"].clone(), "k": a["k"].transpose(1, 2).contiguous().transpose(1, 2)}
    run(b, axes, norm="rms_all", pairing=pairing, q_out=b["q"], k_out=b["k"])
    assert torch.equal(b["q"], want[0]) and torch.equal(b["k"], want[1])


@pytest.mark.parametrize("d,heads", [(128, 48), (64, 130), (128, 25)])
def test_many_heads_past_the_caches(cuda, d, heads):
    """The same at 192 MiB a call and more, in place, against the tokens in calls of their own."""
    tokens = (192 << 20) // (8 * d * heads) + 9
    print(f"case {heads} x {tokens} x {d}", flush=True)
    a = make(19, 1, heads, tokens, d, norm="rms_all")
    axes = recap_amd.rotary_axes((1, 1, tokens), CHANNELS[d], device=cuda)
    whole = run(a, axes, norm="rms_all")
    for first in (0, tokens // 2, tokens - 9):
        part = {m: v[:, :, first:first + 9] if len(m) == 1 else v for m, v in a.items()}
        got = run(part, (*axes[:2], axes[2][first:first + 9]), norm="rms_all")
        assert all(torch.equal(x, y[:, :, first:first + 9]) for x, y in zip(got, whole))
    run(a, axes, norm="rms_all", q_out=a["q"], k_out=a["k"])
    assert torch.equal(a["q"], whole[0]) and torch.equal(a["k"], whole[1])
