"""norm_modulate, gated_residual and gated_residual_norm on the GPU against their definitions in
64 bits: types, norms, broadcasts, widths from 1 to beyond the register kernel's, strides and
alignments, in place, on other streams and in graphs."""

import itertools

import pytest
import torch

from around_util import check, residual
from recap_amd import kernels as K

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [(BF, BF, BF), (BF, BF, F32), (FP, FP, FP), (FP, FP, F32), (F32, BF, F32), (F32, FP, FP),
         (F32, F32, F32)]  # stream; branch and output; modulation


def make(seed, batch, tokens, width, types=(BF, BF, F32), mod="sample", affine=True, wtype=None):
    """A call's tensors: the stream with a mean and channels of other sizes, modulation slices
    of one embedding, weights around one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    stream, t, m = types
    t_w = wtype or t
    out = dict(x=((2 * rand(batch, tokens, width) + 0.5) * rand(width).exp()).to(stream),
               branch=(rand(batch, tokens, width) - 0.25).to(t))
    if mod != "none":
        lead = {"width": (), "sample": (batch,), "sample1": (batch, 1), "token": (batch, tokens),
                "one": (1, 1), "tokens1": (1, tokens)}[mod]
        emb = (0.4 * rand(*lead, 3, width)).to(m)
        out.update((n, emb[..., i, :]) for i, n in enumerate(("gate", "scale", "shift")))
    if affine:
        out.update((n, (base + 0.3 * rand(width)).to(t_w)) for n, base in
                   (("weight", 1), ("bias", 0), ("branch_weight", 1), ("branch_bias", 0)))
    return out


def pick(a, *names):
    return {n: a[n] for n in names if n in a}


def run_pre(a, norm, dtype=None, **more):
    return K.norm_modulate(a["x"], a.get("scale"), a.get("shift"), norm=norm, dtype=dtype,
                           **pick(a, "weight", "bias"), **more)


def run_gate(a, post, **more):
    named = pick(a, "branch_weight", "branch_bias") if post else {}
    return K.gated_residual(a["x"], a["branch"], a.get("gate"), branch_norm=post, **named, **more)


def run_both(a, norm, post, **more):
    named = pick(a, "weight", "bias", *(("branch_weight", "branch_bias") if post else ()))
    return K.gated_residual_norm(a["x"], a["branch"], a.get("gate"), a.get("scale"),
                                 a.get("shift"), norm=norm, branch_norm=post, **named, **more)


def check_all(a, norm, post, label):
    """The three calls on the same tensors against the definitions."""
    print(f"case {label} {norm} {post} {tuple(a['x'].shape)}", flush=True)
    t = a["branch"].dtype
    _, want = residual(a["x"], None, None, a.get("scale"), a.get("shift"), kind=norm,
                       **pick(a, "weight", "bias"))
    y = run_pre(a, norm, t)
    assert y.dtype == t
    check(y, want, f"{label} norm_modulate")
    named = pick(a, "branch_weight", "branch_bias") if post else {}
    r_want, y_want = residual(a["x"], a["branch"], a.get("gate"), a.get("scale"), a.get("shift"),
                              kind=norm, post=post, **named, **pick(a, "weight", "bias"))
    r = run_gate(a, post)
    assert r.dtype == a["x"].dtype
    check(r, r_want, f"{label} gated_residual")
    r2, y = run_both(a, norm, post)
    check(y, y_want, f"{label} gated_residual_norm")
    assert torch.equal(r, r2), f"{label}: the two calls' residuals differ"


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("norm,post", list(itertools.product(("layer", "rms"), (None, "rms", "layer"))))
def test_types_and_norms(cuda, types, norm, post):
    check_all(make(1, 2, 19, 200, types), norm, post, f"{types}")


@pytest.mark.parametrize("mod", ["none", "width", "sample", "sample1", "token", "one", "tokens1"])
@pytest.mark.parametrize("wtype", [BF, F32])
def test_broadcasts(cuda, mod, wtype):
    check_all(make(2, 3, 11, 136, (BF, BF, F32), mod, wtype=wtype), "layer", "rms", f"{mod} {wtype}")


@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 31, 64, 65, 127, 128, 136, 511, 512, 520, 1000, 1001,
                                   1155, 1536, 1920, 2047, 2048, 2056, 4096, 4099, 5120, 8184, 8192,
                                   8193, 8200, 12288, 20001])
@pytest.mark.parametrize("types", [(BF, BF, F32), (F32, F32, F32), (F32, FP, FP)], ids=str)
def test_widths(cuda, width, types):
    check_all(make(3, 1, 5, width, types, "sample1"), "layer", "rms", f"width {width}")
    check_all(make(4, 2, 3, width, types, "token", affine=False), "rms", None, f"width {width}")


@pytest.mark.parametrize("batch,tokens", [(1, 1), (1, 2), (3, 1), (2, 77), (1, 257), (5, 1031), (1, 9001)])
@pytest.mark.parametrize("width", [64, 192, 1536])
def test_row_counts(cuda, batch, tokens, width):
    check_all(make(5, batch, tokens, width), "rms", "layer", f"{batch}x{tokens}")


@pytest.mark.parametrize("names", [(), ("gate",), ("scale",), ("shift",), ("gate", "shift"),
                                   ("scale", "weight"), ("bias",), ("branch_bias", "gate"),
                                   ("branch_weight", "scale", "shift")])
def test_optional_vectors(cuda, names):
    a = make(6, 2, 9, 264)
    a = pick(a, "x", "branch", *names)
    check_all(a, "layer", "layer", f"only {names}")


@pytest.mark.parametrize("width", [64, 520, 1001])
@pytest.mark.parametrize("types", [(BF, BF, BF), (F32, BF, F32), (F32, F32, F32)], ids=str)
def test_strides_and_alignment(cuda, width, types):
    """Slices with odd offsets and pitches, transposed batches, channel strides, expanded
    inputs, and outputs given as such slices; what lies beside an output stays as it was."""
    a = make(7, 3, 7, width, types, "token")
    plain = {n: v.clone() for n, v in a.items()}

    def shifted(v, by, pad):
        buf = torch.zeros(*v.shape[:-1], v.shape[-1] + pad, dtype=v.dtype, device=v.device)
        view = buf[..., by:by + v.shape[-1]]
        view.copy_(v)
        return view

    ways = {"odd offset": lambda v: shifted(v, 1, 3), "odd pitch": lambda v: shifted(v, 0, 1),
            "aligned pitch": lambda v: shifted(v, 8, 16),
            "token major": lambda v: v.transpose(0, 1).contiguous().transpose(0, 1)
            if v.ndim == 3 else v,
            "channel stride": lambda v: torch.stack((v, v), -1)[..., 0]}
    want_y = run_pre(plain, "layer", types[1])
    want = run_both(plain, "layer", "rms")
    for label, way in ways.items():
        print(f"case {label} width {width} {types}", flush=True)
        b = {n: way(v) for n, v in plain.items()}
        assert torch.equal(run_pre(b, "layer", types[1]), want_y), label
        got = run_both(b, "layer", "rms")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), label
        if label == "channel stride":
            continue
        outs = [way(torch.full_like(v, 7.0)) for v in want]
        rings = [o._base if o._base is not None else o for o in outs]
        before = [r.clone() for r in rings]
        run_both(b, "layer", "rms", out=outs[0], norm_out=outs[1])
        for o, w, ring, old in zip(outs, want, rings, before):
            assert torch.equal(o, w), label
            written = torch.zeros_like(ring, dtype=torch.bool)
            torch.as_strided(written, o.shape, o.stride(), o.storage_offset()).fill_(True)
            assert torch.equal(ring[~written], old[~written]), label
    b = {n: v[:1].expand(3, *v.shape[1:]) if v.ndim == 3 else v for n, v in plain.items()}
    got, one = run_both(b, "rms", None), run_both({n: v[:1] if v.ndim == 3 else v
                                                   for n, v in plain.items()}, "rms", None)
    for o, w in zip(got, one):
        assert torch.equal(o, w.expand_as(o))


@pytest.mark.parametrize("width", [192, 1001, 1536, 9000])
def test_in_place(cuda, width):
    """Outputs over their own inputs give what separate outputs give."""
    for types in [(BF, BF, BF), (F32, FP, F32)]:
        a = make(8, 2, 33, width, types)
        want_r = run_gate(a, "rms")
        x = a["x"].clone()
        assert run_gate({**a, "x": x}, "rms", out=x) is x and torch.equal(x, want_r)
        want = run_both(a, "layer", "layer")
        x, br = a["x"].clone(), a["branch"].clone()
        run_both({**a, "x": x, "branch": br}, "layer", "layer", out=x, norm_out=br)
        assert torch.equal(x, want[0]) and torch.equal(br, want[1])
        if types[0] == types[1]:
            want_y, x = run_pre(a, "layer"), a["x"].clone()
            run_pre({**a, "x": x}, "layer", out=x)
            assert torch.equal(x, want_y)


@pytest.mark.parametrize("width", [256, 1001])
def test_values_that_are_not_numbers(cuda, width):
    """Infinities and NaN reach the outputs of their own rows only, as the formula has it; zero
    and constant rows stay finite."""
    a = make(9, 1, 6, width, (BF, BF, BF), "none", affine=False)
    clean = [v.clone() for v in run_both(a, "layer", None)]
    a["x"][0, 1, 3] = float("inf")
    a["x"][0, 3, width - 1] = float("nan")
    a["x"][0, 4] = 0.0
    a["branch"][0, 4] = 0.0
    a["x"][0, 5] = 3.0
    a["branch"][0, 5] = 1.0
    r, y = run_both(a, "layer", None)
    y_rms = run_both(a, "rms", None)[1]
    for row in (0, 2):
        assert torch.equal(r[0, row], clean[0][0, row]) and torch.equal(y[0, row], clean[1][0, row])
    assert r[0, 1, 3] == float("inf") and torch.isnan(y[0, 1]).all()
    rms_row = y_rms[0, 1]   # inf / inf at its own place, finite / inf = 0 elsewhere
    assert torch.isnan(rms_row[3]) and rms_row.nan_to_num(0.0).abs().max() == 0
    assert torch.isnan(r[0, 3, width - 1]) and torch.isnan(y[0, 3]).all() and torch.isnan(y_rms[0, 3]).all()
    assert (y[0, 4] == 0).all() and (y_rms[0, 4] == 0).all()
    assert (y[0, 5] == 0).all()


@pytest.mark.parametrize("width", [16383, 16384, 16385, 20001, 24576, 24577, 32760, 32768, 32769])
@pytest.mark.parametrize("types", [(BF, BF, F32), (FP, FP, FP), (F32, F32, F32)], ids=str)
def test_widths_at_the_registers_end(cuda, width, types):
    """16,384 channels of an fp32 stream and 32,768 of a 16-bit one are what 1024 lanes hold."""
    check_all(make(33, 1, 3, width, types, "sample1"), "layer", "rms", f"width {width}")
    a = make(34, 2, 5, width, types, "token", affine=False)
    check_all(a, "rms", "layer", f"width {width}")
    want, x, branch = run_both(a, "rms", "layer"), a["x"].clone(), a["branch"].clone()
    run_both({**a, "x": x, "branch": branch}, "rms", "layer", out=x, norm_out=branch)
    assert torch.equal(x, want[0]) and torch.equal(branch, want[1])


@pytest.mark.parametrize("width", [14, 15, 28, 61, 448, 832, 960, 1001, 1920, 3840, 7168, 8064])
@pytest.mark.parametrize("types", [(BF, BF, BF), (FP, FP, FP), (F32, FP, FP), (F32, F32, F32)], ids=str)
def test_rows_of_equal_values(cuda, width, types):
    """LayerNorm of a row of equal values is 0 exactly, the shift with one.  The values have few bits,
    so that sums are exact in fp32 in any order, and the widths are such that most of the values
    times a rounded 1 / width miss the mean."""
    x = torch.tensor([3.0, 1000.0, -77.0, 0.84375, 1960.0, 0.0], device=cuda)[None, :, None]
    x = x.expand(2, 6, width).to(types[0]).contiguous()
    shift = torch.linspace(-1, 1, width, device=cuda).to(types[2])
    assert not K.norm_modulate(x, dtype=types[1]).any()
    y = K.norm_modulate(x, None, shift, dtype=types[1])
    assert torch.equal(y, shift.to(types[1]).expand_as(y))
    branch = x.to(types[1])
    r, y = K.gated_residual_norm(x, branch)
    assert torch.equal(r, (2 * x.double()).to(types[0])) and not y.any()
    assert torch.equal(K.gated_residual(x, branch, branch_norm="layer"), x)


def test_a_large_mean(cuda):
    """A row whose mean is 1000 times its deviation: the variance is taken about the mean."""
    a = make(10, 2, 9, 2048, (F32, F32, F32), "none", affine=False)
    a["x"] = 1000.0 + 0.5 * torch.randn(2, 9, 2048, device=cuda)
    check_all(a, "layer", None, "large mean")


@pytest.mark.parametrize("post", ["rms", "layer"])
def test_the_widest_rows(cuda, post):
    """2^24 channels, fp32, with a norm of the branch and one of the sum: rows of equal values, rows
    of values up to 1e17, whose squares' sum is past fp32's range, and ordinary ones.  With sums in
    64 bits an element is off by its own roundings only.  A norm has three (the difference, the root,
    their product), the sum one more of the sum's size: 12 half steps cover them.  The second norm
    adds its three, and the first's errors through its element, mean and deviation: 24."""
    width = 1 << 24
    g = torch.Generator(device="cuda").manual_seed(40)
    x = torch.randn(1, 3, width, generator=g, device="cuda")
    x[0, 0] = 1.1
    x[0, 1].clamp_(-6, 6).mul_(1.6e16)
    f = x * 1.0
    for kind in ("rms", "layer"):
        print(f"case {post} {kind}", flush=True)
        r, y = K.gated_residual_norm(x, f, norm=kind, branch_norm=post)
        y1 = K.norm_modulate(x, norm=kind)
        for row in range(3):
            v = x[0, row].double()
            mean = v.mean() if kind == "layer" else v.new_zeros(())
            dev = ((v - mean).square().mean() + 1e-6).sqrt()
            limit = 12 * 2.0 ** -24 * (v.abs() / dev + 1)
            assert ((y1[0, row].double() - (v - mean) / dev).abs() <= limit).all(), (kind, row)
            m = v.mean() if post == "layer" else v.new_zeros(())
            d = ((v - m).square().mean() + 1e-6).sqrt()
            sizes = v.abs() + v.abs() / d + 1
            sum_ = v + (v - m) / d
            assert ((r[0, row].double() - sum_).abs() <= 12 * 2.0 ** -24 * sizes).all(), (kind, row)
            mean = sum_.mean() if kind == "layer" else v.new_zeros(())
            dev = ((sum_ - mean).square().mean() + 1e-6).sqrt()
            limit = 24 * 2.0 ** -24 * (sizes / dev + 1)
            assert ((y[0, row].double() - (sum_ - mean) / dev).abs() <= limit).all(), (kind, row)


def test_one_channel_with_another_stride(cuda):
    """Rows of one channel, whose stride means nothing (transposed from [batch, 1, tokens])."""
    x = torch.randn(2, 1, 5, device=cuda).transpose(1, 2)
    scale = torch.randn(1, 3, device=cuda)[:, ::3]
    assert x.stride() == (5, 1, 5)
    want = K.gated_residual_norm(x.contiguous(), x.contiguous(), None, scale.clone(), norm="rms")
    got = K.gated_residual_norm(x, x, None, scale, norm="rms")
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty(cuda):
    for shape in [(0, 5, 64), (2, 0, 64)]:
        x = torch.zeros(shape, dtype=BF, device=cuda)
        assert K.norm_modulate(x).shape == shape
        assert all(o.shape == shape for o in K.gated_residual_norm(x, x))
        assert K.gated_residual(x, x).shape == shape


def test_refusals_on_the_gpu(cuda):
    x = torch.zeros(1, 4, 64, dtype=BF, device=cuda)
    with pytest.raises(ValueError, match="GPU"):
        K.gated_residual(x, x.cpu())
    with pytest.raises(ValueError, match="gradient"):
        K.norm_modulate(x, weight=torch.ones(64, dtype=BF, device=cuda, requires_grad=True))
    with torch.no_grad():
        K.norm_modulate(x, weight=torch.ones(64, dtype=BF, device=cuda, requires_grad=True))
    with pytest.raises(ValueError, match="overlaps"):
        K.gated_residual_norm(x, x.clone(), out=x, norm_out=x)
    with pytest.raises(ValueError, match="overlaps"):
        K.gated_residual(x[:, 1:], x[:, 1:].clone(), out=x[:, :3])
    with pytest.raises(ValueError, match="expected"):
        K.norm_modulate(x, out=torch.empty(1, 4, 64, device=cuda))


def test_another_stream_and_two_at_once(cuda):
    """Calls on two streams, their own inputs made there, equal those on the default stream."""
    cases = [make(11 + i, 2, 500, 1536) for i in range(2)]
    torch.cuda.synchronize()
    want = [run_both(a, "layer", "rms") for a in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run_both(cases[i], "layer", "rms"))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for g in runs:
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_captured_and_replayed(cuda):
    """A captured chain of the calls, in place, replayed on new inputs with eager calls between."""
    a = make(13, 2, 130, 1536)
    fresh = [make(20 + i, 2, 130, 1536) for i in range(4)]

    def chain(a):
        y = run_pre(a, "layer", BF)
        r, z = K.gated_residual_norm(a["x"], y, a["gate"], a["scale"], a["shift"], norm="rms")
        return K.gated_residual(r, z, a["gate"], branch_norm="layer")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(a)
    for f in fresh:
        want = chain(f)
        torch.cuda.synchronize()
        for n, v in f.items():
            a[n].copy_(v)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_offsets_beyond_32_bits(cuda):
    """Rows whose element offsets pass 2^31 and 2^32: the last rows equal the same rows alone."""
    batch, tokens, width = 1, 2_200_000, 2048
    x = torch.zeros(batch, tokens, width, dtype=BF, device=cuda)
    assert x.numel() > 2 ** 32
    tail = make(30, 1, 9, width, (BF, BF, BF), "none", affine=False)
    x[:, -9:] = tail["x"]
    want = K.norm_modulate(tail["x"])
    got = K.norm_modulate(x, out=x)
    assert torch.equal(got[:, -9:], want) and not got[:, :-9].any()


def test_more_rows_than_one_launch(cuda):
    """Rows beyond a launch's 2^20 workgroups (of 256 rows each at this width)."""
    rows = (1 << 28) + 1000
    x = torch.zeros(1, rows, 8, dtype=BF, device=cuda)
    tail = make(31, 1, 700, 8, (BF, BF, BF), "none", affine=False)["x"]
    x[:, -700:] = tail
    want = K.gated_residual(tail, tail, branch_norm="rms")
    got = K.gated_residual(x, x.clone(), branch_norm="rms", out=x)
    assert torch.equal(got[:, -700:], want) and not got[:, :-700].any()


@pytest.mark.parametrize("types", [(BF, BF, F32), (F32, FP, F32), (F32, F32, F32)], ids=str)
@pytest.mark.parametrize("batch,tokens,width", [(1, 40000, 1536), (3, 90001, 100), (2, 30011, 520),
                                                (3, 9001, 700), (2, 9007, 1155), (2, 45001, 2048),
                                                (1, 9001, 3001), (2, 2001, 8192)])
def test_large_calls_equal_small_ones(cuda, types, batch, tokens, width):
    """A call large enough to load past the caches, or to take several rows a lane, gives each
    row what a call of its own does."""
    a = make(32, batch, tokens, width, types)
    whole, pre, gate = run_both(a, "layer", "rms"), run_pre(a, "rms", types[1]), run_gate(a, None)
    for rows in (slice(0, 3), slice(tokens // 2, tokens // 2 + 9), slice(tokens - 5, tokens)):
        part = {n: v[:, rows] if v.ndim == 3 else v for n, v in a.items()}
        got = run_both(part, "layer", "rms")
        assert torch.equal(got[0], whole[0][:, rows]) and torch.equal(got[1], whole[1][:, rows])
        assert torch.equal(run_pre(part, "rms", types[1]), pre[:, rows])
        assert torch.equal(run_gate(part, None), gate[:, rows])


@pytest.mark.parametrize("types,width", [
    ((BF, BF, F32), 256), ((BF, BF, F32), 768), ((BF, BF, F32), 1536), ((FP, FP, FP), 1155),
    ((F32, FP, F32), 128), ((F32, FP, F32), 512), ((F32, BF, F32), 768), ((F32, BF, F32), 1024),
    ((F32, F32, F32), 128), ((F32, F32, F32), 500), ((F32, F32, F32), 768), ((F32, F32, F32), 1001)], ids=str)
def test_rows_past_the_caches_equal_small_calls(cuda, types, width):
    """320 MiB of normalised rows and more are stored past the caches: every number of chunks and rows
    a lane holds, against the same rows in calls of their own, and in place."""
    size = 4 if types[1] == F32 else 2
    tokens = (320 << 20) // (width * size) // 2 * 2 + 7
    print(f"case {types} {tokens} x {width}", flush=True)
    a = make(35, 1, tokens, width, types)
    whole, pre = run_both(a, "layer", None), run_pre(a, "rms", types[1])
    posted = run_both(a, "rms", "layer")
    for rows in (slice(0, 70), slice(tokens // 2, tokens // 2 + 9), slice(tokens - 71, tokens)):
        part = {n: v[:, rows] if v.ndim == 3 and v.shape[1] > 1 else v for n, v in a.items()}
        for got, want in ((run_both(part, "layer", None), whole), (run_both(part, "rms", "layer"), posted)):
            assert torch.equal(got[0], want[0][:, rows]) and torch.equal(got[1], want[1][:, rows])
        assert torch.equal(run_pre(part, "rms", types[1]), pre[:, rows])
    del posted, pre
    run_both(a, "layer", None, out=a["x"], norm_out=a["branch"])
    assert torch.equal(a["x"], whole[0]) and torch.equal(a["branch"], whole[1])


@pytest.mark.parametrize("width", [1, 5, 7, 32769, 40001])
@pytest.mark.parametrize("types", [(BF, BF, BF), (F32, FP, F32), (F32, F32, F32)], ids=str)
def test_in_place_beyond_the_registers(cuda, width, types):
    """The rows that a workgroup reads again for each sum, over their own inputs."""
    a = make(36, 2, 33, width, types)
    for norm, post in (("layer", "layer"), ("rms", None)):
        want = run_both(a, norm, post)
        x, br = a["x"].clone(), a["branch"].clone()
        run_both({**a, "x": x, "branch": br}, norm, post, out=x, norm_out=br)
        assert torch.equal(x, want[0]) and torch.equal(br, want[1])
        want, x = run_gate(a, post), a["x"].clone()
        assert torch.equal(run_gate({**a, "x": x}, post, out=x), want)
        if types[0] == types[1]:
            want, x = run_pre(a, norm), a["x"].clone()
            assert torch.equal(run_pre({**a, "x": x}, norm, out=x), want)


@pytest.mark.parametrize("width", [3, 5])
def test_more_short_rows_than_workgroups(cuda, width):
    """Rows under a chunk, more than a launch's 2^20 workgroups: a workgroup takes several."""
    a = make(37, 2, (1 << 20) + 300, width, (BF, BF, F32))
    tokens = a["x"].shape[1]
    whole, pre = run_both(a, "layer", "rms"), run_pre(a, "rms")
    x, br = a["x"].clone(), a["branch"].clone()
    run_both({**a, "x": x, "branch": br}, "layer", "rms", out=x, norm_out=br)
    assert torch.equal(x, whole[0]) and torch.equal(br, whole[1])
    for rows in (slice(0, 40), slice(tokens - 700, tokens - 600), slice(tokens - 40, tokens)):
        part = {n: v[:, rows] if v.ndim == 3 else v for n, v in a.items()}
        got = run_both(part, "layer", "rms")
        assert torch.equal(got[0], whole[0][:, rows]) and torch.equal(got[1], whole[1][:, rows])
        assert torch.equal(run_pre(part, "rms"), pre[:, rows])
