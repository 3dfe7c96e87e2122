"""AttentionBlock on the GPU: the whole attention half of a block, refresh then sparse steps,
against its parts one by one (bit for bit) and against 64 bits around the oracle's attention."""

import pytest
import torch

import oracle as O
import recap_amd
from around_util import check, qk, residual
from gpu_util import SMALL, metrics
from recap_amd import EXACT, REFRESH, SPARSE, OperatorConfig, kernels as K
from recap_amd.layout import Layout, SparseGeometry, hilbert_permutation

pytestmark = pytest.mark.gpu

CHANNELS = {64: (16, 24, 24), 128: (44, 42, 42)}


def build(wl, cuda, qk_norm, stream, batch, width=320, seed=0):
    perm = hilbert_permutation(wl.grid)
    layout = Layout.from_permutation(perm, text_tokens=wl.text_tokens, text_first=wl.text_first)
    op = recap_amd.Operator.build(OperatorConfig(head_density=wl.density),
                                  SparseGeometry.build(layout, 128), n_layers=1)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    inner, dtype = wl.heads * wl.dim, wl.dtype
    w = {n: (rand(*s) * s[1] ** -0.5).to(dtype) for n, s in
         (("q", (inner, width)), ("k", (inner, width)), ("v", (inner, width)), ("o", (width, inner)))}
    linear = {n: (lambda y, m=m: y @ m.T) for n, m in w.items()}
    extent = inner if qk_norm == "rms_all" else wl.dim
    block = recap_amd.AttentionBlock(
        op, 0, wl.heads, linear["q"], linear["k"], linear["v"], linear["o"],
        axes=recap_amd.rotary_axes(wl.grid, CHANNELS[wl.dim], device=cuda), qk_norm=qk_norm,
        q_weight=(1 + 0.2 * rand(extent)).to(dtype), k_weight=(1 + 0.2 * rand(extent)).to(dtype),
        branch_norm="rms", branch_weight=(1 + 0.2 * rand(width)).to(dtype), next_norm="rms", dtype=dtype)
    emb = 0.3 * rand(batch, 5, width)
    steps = [rand(batch, wl.tokens, width)]
    for _ in range(2):
        steps.append(steps[-1] + 0.02 * rand(batch, wl.tokens, width))
    return block, w, [emb[:, i:i + 1] for i in range(5)], [s.to(stream) for s in steps], perm


@pytest.mark.parametrize("name,qk_norm,stream,batch", [
    ("text-last-d128", "rms", torch.bfloat16, 1), ("text-first-ragged", "layer", torch.float32, 2),
    ("video-ragged-d128", "rms_all", torch.float32, 1)])
def test_block_steps(cuda, name, qk_norm, stream, batch):
    wl = SMALL[name]
    block, w, mods, steps, perm = build(wl, cuda, qk_norm, stream, batch)
    op = block.operator
    ref = recap_amd.Operator.build(op.config, op.layers[0][0].geometry, n_layers=1)
    oracle = O.OracleOperator(wl.grid, wl.text_tokens, wl.text_first, wl.density, permutation=perm)
    scale, shift, gate, scale2, shift2 = mods
    for step, (x, kind) in enumerate(zip(steps, (REFRESH, SPARSE, SPARSE))):
        print(f"case {name} {qk_norm} step {step} {kind}", flush=True)
        op.begin_step(step, kind)
        ref.begin_step(step, kind)
        r, y = block(x, scale, shift, gate, scale2, shift2)
        # its parts, one by one
        h = K.norm_modulate(x, scale, shift, dtype=wl.dtype)
        q, k, v = ((h @ w[n].T).unflatten(2, (wl.heads, wl.dim)).transpose(1, 2) for n in "qkv")
        qr, kr = K.qk_rotary(q, k, block.axes, offset=op.layout.video_offset, norm=qk_norm,
                             q_weight=block.q_weight, k_weight=block.k_weight)
        out = ref.attend(0, qr, kr, v)
        branch = out.transpose(1, 2).flatten(2) @ w["o"].T
        parts = K.gated_residual_norm(x, branch, gate, scale2, shift2, norm="rms",
                                      branch_norm="rms", branch_weight=block.branch_weight)
        assert torch.equal(r, parts[0]) and torch.equal(y, parts[1])
        # the definitions in 64 bits around the oracle's attention, each part on its own inputs'
        # rounding: queries and keys rounded once as the kernels take them
        exact_q, exact_k = (qk(t, block.axes, offset=op.layout.video_offset, kind=qk_norm,
                               weight=wt)[0].to(wl.dtype)
                            for t, wt in ((q, block.q_weight), (k, block.k_weight)))
        args = (0, exact_q.cpu(), exact_k.cpu(), v.cpu())
        want = (oracle.refresh if kind == REFRESH else oracle.sparse)(*args).to(wl.dtype).to(cuda)
        branch = want.transpose(1, 2).flatten(2) @ w["o"].T
        (er, _), (ey, _) = residual(x, branch, gate, scale2, shift2, kind="rms", post="rms",
                                    branch_weight=block.branch_weight)
        for label, got, exact in (("residual", r, er), ("normed", y, ey)):
            _, cos = metrics(got, exact)
            assert cos >= 0.999, (label, cos)


def test_block_exact_step_and_text_length(cuda):
    """An EXACT step, and a per-prompt text length that moves the video's first token."""
    wl = SMALL["text-first-ragged"]
    block, w, mods, steps, _ = build(wl, cuda, "rms", torch.bfloat16, 1)
    op = block.operator
    op.begin_step(0, EXACT)
    x = steps[0]
    long = block(x, *mods)
    op.layout.text_tokens -= 100   # the prompt lost its first 100 tokens
    op.layout._gather_cache.clear()
    q = torch.randn(1, wl.heads, wl.tokens - 100, wl.dim, device=cuda).to(wl.dtype)
    h = K.norm_modulate(x[:, 100:], mods[0], mods[1], dtype=wl.dtype)
    seen = {}
    attend = op.attend
    op.attend = lambda layer, query, key, value: seen.update(q=query) or attend(layer, query, key, value)
    short = block(x[:, 100:], *mods)
    q = (h @ w["q"].T).unflatten(2, (wl.heads, wl.dim)).transpose(1, 2)
    want = K.qk_rotary(q, None, block.axes, offset=wl.text_tokens - 100, norm="rms",
                       q_weight=block.q_weight)[0]
    assert torch.equal(seen["q"], want)
    assert short[0].shape[1] == wl.tokens - 100 and torch.isfinite(short[1]).all()
    assert torch.isfinite(long[1]).all()


@pytest.mark.parametrize("call", [
    lambda x, b: K.norm_modulate(x, out=x), lambda x, b: K.gated_residual(x, b, out=x),
    lambda x, b: K.gated_residual_norm(b, x, norm_out=x),
    lambda x, b: K.gated_residual_norm(x, b[..., ::2].repeat_interleave(2, -1), b.new_zeros(1, 128)[:, ::2],
                                       out=x),
    lambda x, b: K.qk_rotary(x[None], None, norm="rms", q_out=x[None]),
    lambda x, b: K.qk_rotary(b[None], x[None], norm="rms", k_out=x[None])])
def test_in_place_is_seen_by_autograd(cuda, call):
    """A tensor that a graph saved, then given as an output: the backward pass raises instead of
    giving the gradient of other values.  Outputs that a call makes count no change."""
    x, b = (torch.randn(2, 5, 64, device=cuda).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(64, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    loss = (w * x).sum()
    with torch.no_grad():
        call(x, b)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        call(x, b)
    assert K.norm_modulate(x)._version == 0


@pytest.mark.parametrize("name,qk_norm", [("text-first-ragged", "rms"), ("text-last-d128", "rms_all")])
def test_block_outputs_at_another_text_length(cuda, name, qk_norm):
    """After a prompt's text length changed, an EXACT step's outputs are its parts' one by one, and
    those of the 64-bit definition around the same attention output."""
    import torch.nn.functional as F
    wl = SMALL[name]
    block, w, mods, steps, _ = build(wl, cuda, qk_norm, torch.bfloat16, 1)
    op = block.operator
    op.begin_step(0, EXACT)
    cut = wl.text_tokens // 2
    op.layout.text_tokens -= cut
    op.layout._gather_cache.clear()
    x = steps[0][:, cut:] if wl.text_first else steps[0][:, :-cut]
    scale, shift, gate, scale2, shift2 = mods
    r, y = block(x, *mods)
    h = K.norm_modulate(x, scale, shift, dtype=wl.dtype)
    q, k, v = ((h @ w[n].T).unflatten(2, (wl.heads, wl.dim)).transpose(1, 2) for n in "qkv")
    q, k = K.qk_rotary(q, k, block.axes, offset=op.layout.video_offset, norm=qk_norm,
                       q_weight=block.q_weight, k_weight=block.k_weight)
    branch = F.scaled_dot_product_attention(q, k, v).transpose(1, 2).flatten(2) @ w["o"].T
    parts = K.gated_residual_norm(x, branch, gate, scale2, shift2, norm="rms", branch_norm="rms",
                                  branch_weight=block.branch_weight)
    assert torch.equal(r, parts[0]) and torch.equal(y, parts[1])
    want = residual(x, branch, gate, scale2, shift2, kind="rms", post="rms",
                    branch_weight=block.branch_weight)
    check(r, want[0], "residual")
    check(y, want[1], "normed")


def test_block_norms_with_their_own_eps(cuda):
    """eps, qk_eps and next_eps each reach their own norms."""
    wl = SMALL["video-ragged-d128"]
    block, w, mods, steps, _ = build(wl, cuda, "rms", torch.bfloat16, 1)
    block.eps, block.qk_eps, block.next_eps = 0.3, 0.02, 0.1
    block.operator.begin_step(0, EXACT)
    seen, attend = {}, block.operator.attend
    block.operator.attend = lambda layer, *qkv: seen.update(qkv=qkv, out=attend(layer, *qkv)) or seen["out"]
    x = steps[0]
    r, y = block(x, *mods)
    h = K.norm_modulate(x, mods[0], mods[1], eps=0.3)
    q, k = ((h @ w[n].T).unflatten(2, (wl.heads, wl.dim)).transpose(1, 2) for n in "qk")
    for got, t, weight in ((seen["qkv"][0], q, block.q_weight), (seen["qkv"][1], k, block.k_weight)):
        check(got, qk(t, block.axes, kind="rms", weight=weight, eps=0.02), "queries and keys")
    branch = seen["out"].transpose(1, 2).flatten(2) @ w["o"].T
    want = residual(x, branch, *mods[2:], kind="rms", post="rms", branch_weight=block.branch_weight, eps=0.1)
    check(r, want[0], "residual")
    check(y, want[1], "normed")


@pytest.mark.parametrize("text_first", [False, True])
@pytest.mark.parametrize("heads,d", [(3, 128), (2, 64)])
@pytest.mark.parametrize("grid", [(3, 5, 10), (3, 15, 20)], ids=str)
def test_two_streams_in_one_sequence(cuda, text_first, heads, d, grid):
    """A block whose text tokens have projections and norms of their own: each stream's queries and
    keys go into its part of the joint sequence, and its part of the attention's output into its own
    residual stream.  A video of at most two blocks may leave rows of a sparse call without a tail,
    which the reference's merge makes NaN: such rows stay NaN and touch no others."""
    text, width, b = 77, 192, 2
    video = grid[0] * grid[1] * grid[2]
    layout = Layout.from_permutation(hilbert_permutation(grid), text_tokens=text, text_first=text_first)
    op = recap_amd.Operator.build(OperatorConfig(head_density=0.5), SparseGeometry.build(layout, 128), n_layers=1)
    axes = recap_amd.rotary_axes(grid, CHANNELS[d], device=cuda)
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    dtype, inner = torch.bfloat16, heads * d
    first = layout.video_offset
    parts = {"video": slice(first, first + video),
             "text": slice(0, text) if text_first else slice(video, video + text)}
    streams = {n: rand(b, video if n == "video" else text, width).to(dtype) for n in parts}
    w = {n: {m: (rand(*s) * s[1] ** -0.5).to(dtype) for m, s in
             (("q", (inner, width)), ("k", (inner, width)), ("v", (inner, width)), ("o", (width, inner)))}
         for n in parts}
    norms = {n: [(1 + 0.2 * rand(d)).to(dtype) for _ in "qk"] for n in parts}
    mods = {n: [0.3 * rand(b, 1, width) for _ in range(5)] for n in parts}

    joint = [torch.full((b, video + text, heads, d), 7.0, dtype=dtype, device=cuda).transpose(1, 2)
             for _ in "qkv"]
    split = {}
    for n, at in parts.items():
        h = K.norm_modulate(streams[n], mods[n][0], mods[n][1])
        q, k, v = ((h @ w[n][m].T).unflatten(2, (heads, d)).transpose(1, 2) for m in "qkv")
        split[n] = q, k
        K.qk_rotary(q, k, axes if n == "video" else None, norm="rms", q_weight=norms[n][0],
                    k_weight=norms[n][1], q_out=joint[0][:, :, at], k_out=joint[1][:, :, at])
        joint[2][:, :, at] = v
    for n, at in parts.items():
        for i in range(2):
            check(joint[i][:, :, at], qk(split[n][i], axes if n == "video" else None, kind="rms",
                                         weight=norms[n][i]), f"{n} {'qk'[i]}")
    for step, kind in enumerate((REFRESH, SPARSE)):
        print(f"case {heads} x {d} text first {text_first} {kind}", flush=True)
        op.begin_step(step, kind)
        out = op.attend(0, *joint).transpose(1, 2)
        for n, at in parts.items():
            branch = out[:, at].flatten(2) @ w[n]["o"].T
            r, y = K.gated_residual_norm(streams[n], branch, *mods[n][2:])
            want = residual(streams[n], branch, *mods[n][2:], kind="layer")
            rows = ~branch.isnan().any(-1)
            assert rows.all() or (video <= 256 and kind == SPARSE and branch[~rows].isnan().all())
            assert r[~rows].isnan().all() and y[~rows].isnan().all()
            for label, got, (exact, bound) in (("residual", r, want[0]), ("normed", y, want[1])):
                check(got[rows], (exact[rows], bound[rows]), f"{n} {label}")
