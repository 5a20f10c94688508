"""Causal attention with a sliding window and sinks against the FP64 oracle: gradients, positions, positions per
sequence, hidden rows, layouts, graphs, streams, the compiled route and the refusals."""

import pytest
import torch

from oracle import attention_oracle as ao
from tests.helpers import NAMES, TOL, make_inputs, run_attention, strided_like_projection

pytestmark = pytest.mark.gpu


def api():
    import kohakufa_cute

    return kohakufa_cute


def native():
    from kohakufa_cute import native as module

    return module


def window_mask(starts, Sq, Sk, window, sinks):
    """[B, 1, Sq, Sk] visibility from the definition."""
    pos = torch.as_tensor(starts, dtype=torch.int64)[:, None, None] + torch.arange(Sq)[None, :, None]
    key = torch.arange(Sk)[None, None, :]
    return ((key <= pos) & ((key > pos - window) | (key < sinks)))[:, None]


def check(actual, q, k, v, dout, mask, scale):
    """(out, dq, dk, dv) against FP64 mathematics: the operator's per-head norm gates, and every element within the
    sum of the roundings behind it.  With u = half a step of the 16-bit type (relative):
      out    u |O| + sum_c u P |V|                              its own rounding; P rounded for the product
      delta  e = sum_d |dO| (u |O| + sum_c u P |V|)             formed from the stored O
      dV     u |dV| + sum_r u P |dO|                            P rounded
      dK     u |dK| + scale sum_r (u |dS| + P e) |Q|            dS rounded; delta's error
      dQ     u |dQ| + scale sum_c (u |dS| + P e) (|K| + max |K|)   the same, keys less a mean key
    FP32 steps (score sums, ex2, normaliser: below 3e-5 relative to the same sums) are covered by a tenth of u more."""
    want = ao.math_reference([t.cpu() for t in (q, k, v)], dout.cpu(), mask, False, scale)
    B, Hq, Sq, D = q.shape
    group = Hq // k.shape[1]
    qd, kd, vd, gd = (t.cpu().double() for t in (q, k, v, dout))
    kd, vd = kd.repeat_interleave(group, 1), vd.repeat_interleave(group, 1)
    c = D**-0.5 if scale is None else scale
    seen = mask.expand(B, Hq, Sq, k.shape[2])
    s = (qd @ kd.transpose(-1, -2) * c).masked_fill(~seen, float("-inf"))
    prob = torch.softmax(s.masked_fill(~seen.any(-1, keepdim=True), 0.0), -1).masked_fill(~seen, 0.0)
    u = 1.1 * torch.finfo(q.dtype).eps / 2
    spread = u * (prob @ vd.abs())
    out = want[0]
    e = (gd.abs() * (u * out.abs() + spread)).sum(-1, keepdim=True)
    ds = prob * (gd @ vd.transpose(-1, -2) - (gd * out).sum(-1, keepdim=True))
    noise = u * ds.abs() + prob * e

    def shared(t):
        return t.reshape(B, Hq // group, group, *t.shape[2:]).sum(2)

    top = kd.abs().amax(2, keepdim=True)
    bounds = (u * out.abs() + spread,
              u * want[1].abs() + abs(c) * (noise @ kd.abs() + noise.sum(-1, keepdim=True) * top),
              u * want[2].abs() + abs(c) * shared(noise.transpose(-1, -2) @ qd.abs()),
              u * want[3].abs() + shared(u * prob.transpose(-1, -2) @ gd.abs()))
    tiny = torch.finfo(q.dtype).smallest_normal  # results below it are rounded in absolute steps, or flushed
    for name, got, exact, bound in zip(NAMES, actual, want, bounds):
        got = got.detach().cpu().double()
        assert bool(torch.isfinite(got).all()), name
        if float(exact.abs().max()) == 0:
            assert float(got.abs().max()) <= float(bound.max()), name
            continue
        far = ((got - exact).abs() - bound - tiny).max()
        assert float(far) <= 0, f"{name}: an element is {float(far):.3e} beyond its roundings"
        # bounds are worst cases; a head's norm averages them
        err = ao.per_head_relative_error(got, exact)
        limit = max(TOL[q.dtype]["norm"], float((bound.norm(dim=(2, 3)) / exact.norm(dim=(2, 3)).clamp_min(1e-300)).max()) / 2)
        assert err < limit, f"{name}: per-head relative error {err:.3e} (limit {limit:.3e})"
    return want


SHAPES = (
    # B, Hq, Hkv, Sq, Sk, D, window, sinks, start
    (1, 4, 2, 300, 300, 128, 64, 4, 0),
    (2, 2, 2, 129, 257, 64, 1, 0, 128),        # every row sees itself only
    (1, 4, 1, 513, 700, 96, 130, 130, 187),    # the sinks reach into the second key tile
    (2, 4, 2, 1025, 1025, 128, 300, 5, 0),     # tiles between the sinks and the window
    (1, 2, 2, 1, 1, 64, 5, 0, 0),              # one token
    (1, 4, 4, 1, 600, 128, 100, 2, 599),       # one row at the end of its keys
    (1, 2, 1, 70, 65, 17, 9, 2, 0),            # more rows than keys, an odd head
    (1, 2, 2, 200, 200, 256, 33, 3, 0),        # a head beyond the pipeline kernels
    (1, 2, 2, 260, 260, 64, 100000, 0, 0),     # a window longer than the sequence: plain causal
    (1, 2, 2, 200, 300, 128, 50, 2, 500),      # behind the keys: the sinks only
    (1, 2, 1, 300, 300, 64, 20, 0, 150),       # the last rows see nothing
    (1, 2, 2, 400, 1000, 64, 128, 1000, 300),  # every key a sink
    (1, 8, 1, 640, 640, 80, 256, 1, 0),
)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients_match_the_oracle(shape, dtype):
    B, Hq, Hkv, Sq, Sk, D, window, sinks, start = shape
    q, k, v, dout = make_inputs(B, Hq, Hkv, Sq, Sk, D, dtype, seed=Sq + Sk + window)
    mask = window_mask([start] * B, Sq, Sk, window, sinks)
    for scale in (None, -0.11):
        actual = run_attention(api().sliding_window_attention, q, k, v, dout, window=window, sinks=sinks,
                               query_start=start, scale=scale)
        if window == 1 and sinks == 0:
            # As with a single key: P = 1 and dS = 0 exactly, so O = V, dQ = dK = 0 and dV = dO summed over the group
            # (the rounding contract's two independent FP32 reductions of dP and delta would invent a few-ulp gradient).
            exact = ao.math_reference([t.cpu() for t in (q, k, v)], dout.cpu(), mask, False, scale)
            assert torch.equal(actual[0].cpu().double(), exact[0]) and torch.equal(actual[3].cpu(), exact[3].to(dtype))
            assert float(actual[1].abs().max()) == 0 and float(actual[2].abs().max()) == 0
        else:
            check(actual, q, k, v, dout, mask, scale)
        blind = ~mask.expand(B, Hq, Sq, Sk).any(-1)
        assert float(actual[0].cpu()[blind].abs().sum()) == 0 and float(actual[1].cpu()[blind].abs().sum()) == 0
        unseen = ~mask.any(2)[:, 0]
        assert all(float(g.cpu().transpose(1, 2)[unseen].abs().sum()) == 0 for g in actual[2:])
    with torch.no_grad():
        inference = api().sliding_window_attention(q, k, v, window=window, sinks=sinks, query_start=start, scale=-0.11)
    if float(actual[0].abs().max()) > 0:
        assert ao.per_head_relative_error(inference.cpu(), actual[0].cpu().double()) < TOL[dtype]["norm"]
    else:
        assert float(inference.abs().max()) == 0
    assert native().device_status(reset=True) == 0


def test_a_zero_scale_averages_the_visible_values():
    q, k, v, dout = make_inputs(1, 2, 1, 150, 150, 64, torch.bfloat16, seed=1)
    actual = run_attention(api().sliding_window_attention, q, k, v, dout, window=40, sinks=2, scale=0.0)
    mask = window_mask([0], 150, 150, 40, 2)
    want = ao.math_reference([t.cpu() for t in (q, k, v)], dout.cpu(), mask, False, 0.0)
    # the output is one rounding (2^-9 of the value) of an average of at most 42 values below about 5
    torch.testing.assert_close(actual[0].cpu().double(), want[0], atol=5 * 2**-9, rtol=2**-7)
    assert float(actual[1].abs().max()) == 0 and float(actual[2].abs().max()) == 0


def test_the_gradient_matches_differences():
    """d(sum(out * dout)) along random directions against central differences of the FP64 definition, at the gradients'
    own 1 % gate (the kernels' gradients are rounded to 16 bits, the differences are formed in 64 bits)."""
    B, Hq, Hkv, S, D, window, sinks = 1, 4, 2, 200, 64, 48, 3
    q, k, v, dout = make_inputs(B, Hq, Hkv, S, S, D, torch.float16, seed=9)
    grads = run_attention(api().sliding_window_attention, q, k, v, dout, window=window, sinks=sinks)[1:]
    mask = window_mask([0], S, S, window, sinks)
    base = [t.cpu().double() for t in (q, k, v)]

    def value(tensors):
        qq, kk, vv = tensors
        kk, vv = (t.repeat_interleave(Hq // Hkv, dim=1) for t in (kk, vv))
        s = (qq @ kk.transpose(-1, -2) * D**-0.5).masked_fill(~mask, float("-inf"))
        return float((torch.softmax(s, -1) @ vv * dout.cpu().double()).sum())

    gen = torch.Generator().manual_seed(4)
    for which, grad in enumerate(grads):
        direction = grad.cpu().double() / grad.cpu().double().norm()
        direction = direction + 0.1 * torch.randn(direction.shape, generator=gen).double() / direction.numel() ** 0.5
        h = 1e-4
        ends = []
        for sign in (1, -1):
            moved = list(base)
            moved[which] = base[which] + sign * h * direction
            ends.append(value(moved))
        want = (ends[0] - ends[1]) / (2 * h)
        got = float((grad.cpu().double() * direction).sum())
        assert abs(got - want) < 0.01 * abs(want)


@pytest.mark.parametrize("case", (
    # Hq, Hkv, Sq, Sk, D, window, sinks, starts
    (4, 2, 300, 900, 128, 128, 4, (600, 100, 0, -40)),
    (8, 2, 1, 700, 128, 256, 4, (699, 5, 0, -1)),
    (8, 8, 4, 515, 64, 100, 0, (511, 1, 700, -3)),
    (8, 1, 3, 1000, 128, 64, 130, (2**31 - 1, 996, 129, -(2**31))),
    (6, 2, 257, 400, 80, 90, 1, (143, 20, 390, 600)),
    (4, 2, 40, 200, 256, 30, 2, (100, 160, 0, 7)),
    (8, 1, 2, 3000, 128, 700, 20, (2998, 1500, 3, 719)),      # sixteen rows per K/V head
    (12, 4, 4, 2000, 64, 5000, 0, (1996, 0, 1000, -2)),       # twelve
    (4, 2, 1, 300, 128, 100, 4, tuple(range(0, 280, 4))),     # seventy sequences
))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_positions_per_sequence(case, dtype):
    """Ragged positions from a device tensor; whatever lies behind a sequence's last position is never looked at."""
    Hq, Hkv, Sq, Sk, D, window, sinks, starts = case
    B = len(starts)
    q, k, v, dout = make_inputs(B, Hq, Hkv, Sq, Sk, D, dtype, seed=Sk + Sq)
    mask = window_mask(starts, Sq, Sk, window, sinks)
    want = ao.math_reference([t.cpu() for t in (q, k, v)], dout.cpu(), mask, False, None)[0]
    garbage = [t.clone() for t in (k, v)]
    for b, start in enumerate(starts):
        end = max(0, min(Sk, start + Sq))
        garbage[0][b, :, end:], garbage[1][b, :, end:] = float("nan"), float("inf")
    at = torch.tensor(starts, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        got = api().sliding_window_attention(q, *garbage, window=window, sinks=sinks, query_start=at)
        again = api().sliding_window_attention(q, *garbage, window=window, sinks=sinks, query_start=at)
    assert torch.equal(got, again) and bool(torch.isfinite(got).all())
    for b in range(B):
        seen = mask[b].any()
        if not seen:
            assert float(got[b].abs().max()) == 0
            continue
        assert ao.per_head_relative_error(got[b:b + 1].cpu(), want[b:b + 1]) < TOL[dtype]["norm"]
    blind = ~mask.any(-1).expand(B, Hq, Sq)
    assert float(got.cpu()[blind].abs().sum()) == 0
    if starts[0] >= 0 and starts[0] < 2**31 - 1:  # the int form is the same call
        one = api().sliding_window_attention(q[:1], k[:1], v[:1], window=window, sinks=sinks, query_start=starts[0])
        torch.testing.assert_close(one, got[:1], atol=TOL[dtype]["elem"], rtol=TOL[dtype]["elem"])
    assert native().device_status(reset=True) == 0


@pytest.mark.parametrize("case", (
    # both sides of the rule that chooses between one cluster per unit and a line of blocks cut over all CTAs, and
    # clusters of several sizes:  Hq, Hkv, Sq, Sk, D, window, sinks, starts
    (4, 2, 1, 160 * 16, 128, 4000, 0, (160 * 16 - 1, -1, 200)),     # the longest that clusters take, and the next
    (4, 2, 1, 160 * 16 + 1, 128, 4000, 0, (160 * 16, -1, 200)),
    (8, 4, 1, 400, 128, 150, 4, tuple(range(-2, 400, 51))),         # 32 units: eight CTAs each
    (8, 4, 1, 400, 128, 150, 4, tuple(range(-2, 400, 41))),         # 40: six
    (8, 8, 1, 300, 128, 150, 4, tuple(range(-2, 300, 28))),         # 88: three
    (8, 8, 1, 300, 128, 150, 4, tuple(range(-2, 300, 9))),          # 272: the line
    (16, 1, 3, 300, 64, 120, 20, tuple(range(-4, 320, 17))),        # three units of 16 rows: 60
    # more rows than a unit has, on both sides of the rule that leaves them to the tensor-memory forward
    (32, 4, 4, 900, 128, 500, 4, (896, 2, -3, 500, 901)),           # 32 rows
    (4, 2, 33, 700, 128, 300, 0, (667, 0, -20, 690)),               # 66: the last unit holds two
    (8, 1, 100, 600, 64, 77, 3, (500, 30, 590)),
    (6, 2, 256, 900, 128, 800, 130, (644, -100)),
    (2, 2, 64, 300, 128, 50, 1, tuple(range(-60, 300, 3))),         # 120 sequences: too many
))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_decoding_of_short_and_full_batches(case, dtype):
    Hq, Hkv, Sq, Sk, D, window, sinks, starts = case
    q, k, v, dout = make_inputs(len(starts), Hq, Hkv, Sq, Sk, D, dtype, seed=Sk + len(starts))
    mask = window_mask(starts, Sq, Sk, window, sinks)
    want = ao.math_reference([t.cpu() for t in (q, k, v)], dout.cpu(), mask, False, None)[0]
    at = torch.tensor(starts, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        got = api().sliding_window_attention(q, k, v, window=window, sinks=sinks, query_start=at)
    for b in range(len(starts)):
        if mask[b].any():
            assert ao.per_head_relative_error(got[b:b + 1].cpu(), want[b:b + 1]) < TOL[dtype]["norm"]
    blind = ~mask.any(-1).expand(len(starts), Hq, Sq)
    assert float(got.cpu()[blind].abs().sum()) == 0
    assert native().device_status(reset=True) == 0


def test_one_new_token_against_a_long_cache():
    """Many CTAs per sequence; the cache is a view of a larger one, [B, S, H, D] in memory."""
    B, Hq, Hkv, Sk, D = 2, 8, 2, 30000, 128
    q, k, v, dout = make_inputs(B, Hq, Hkv, 1, Sk, D, torch.bfloat16, seed=15)
    held = [torch.full((B, Sk + 100, Hkv, D), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    for t, x in zip(held, (k, v)):
        t[:, :Sk] = x.transpose(1, 2)
    views = [t[:, 7:Sk].transpose(1, 2) for t in held]
    for window, sinks in ((20000, 4), (1 << 20, 0), (5, 17)):
        with torch.no_grad():
            got = api().sliding_window_attention(q, *views, window=window, sinks=sinks, query_start=Sk - 8)
        mask = window_mask([Sk - 8] * B, 1, Sk - 7, window, sinks)
        want = ao.math_reference([t.cpu() for t in (q, *views)], dout.cpu(), mask, False, None)[0]
        assert ao.per_head_relative_error(got.cpu(), want) < TOL[torch.bfloat16]["norm"]
    assert native().device_status(reset=True) == 0


@pytest.mark.parametrize("case", (
    # few query tiles, so that a cluster shares a tile's keys:  B, Hq, Hkv, Sq, Sk, D, window, sinks
    (1, 2, 1, 128, 5000, 128, 3000, 4),      # eight CTAs a tile
    (1, 2, 2, 200, 3001, 64, 10000, 300),    # sinks over three key tiles, a query tile that is not full
    (2, 4, 2, 300, 1500, 96, 900, 0),        # channels that the tile pads
    (1, 4, 4, 1000, 1000, 128, 1000, 1),     # tiles at the start see fewer keys than there are CTAs
    (3, 6, 1, 640, 2000, 80, 700, 130),      # two CTAs a tile
))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_few_query_tiles_share_their_keys(case, dtype):
    B, Hq, Hkv, Sq, Sk, D, window, sinks = case
    q, k, v, dout = make_inputs(B, Hq, Hkv, Sq, Sk, D, dtype, seed=Sk)
    for start in (Sk - Sq, 0, Sk - Sq // 2):
        call = dict(window=window, sinks=sinks, query_start=start)
        got = run_attention(api().sliding_window_attention, q, k, v, dout, **call)
        check(got, q, k, v, dout, window_mask([start], Sq, Sk, window, sinks), None)
        again = run_attention(api().sliding_window_attention, q, k, v, dout, **call)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    at = torch.tensor([-Sq - 5, Sk // 2, Sk - 3][:B], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        got = api().sliding_window_attention(q, k, v, window=window, sinks=sinks, query_start=at)
    mask = window_mask(at.tolist(), Sq, Sk, window, sinks)
    want = ao.math_reference([t.cpu() for t in (q, k, v)], dout.cpu(), mask, False, None)[0]
    for b in range(B):
        if mask[b].any():
            assert ao.per_head_relative_error(got[b:b + 1].cpu(), want[b:b + 1]) < TOL[dtype]["norm"]
    blind = ~mask.any(-1).expand(B, Hq, Sq)
    assert float(got.cpu()[blind].abs().sum()) == 0
    assert native().device_status(reset=True) == 0


def test_layouts_give_the_same_result():
    B, Hq, Hkv, S, D, window, sinks = 2, 4, 2, 333, 64, 77, 4
    q, k, v, dout = make_inputs(B, Hq, Hkv, S, S, D, torch.bfloat16, seed=2)
    call = dict(window=window, sinks=sinks)
    want = run_attention(api().sliding_window_attention, q, k, v, dout, **call)
    strided = run_attention(api().sliding_window_attention, *(strided_like_projection(t) for t in (q, k, v)),
                            strided_like_projection(dout), **call)
    wide = torch.zeros(B, Hq, S, 2 * D, device="cuda", dtype=torch.bfloat16)
    wide[..., ::2] = q
    channels = run_attention(api().sliding_window_attention, wide[..., ::2], k, v, dout, **call)
    for a, b, c in zip(want, strided, channels):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_clusters_follow_new_positions():
    B, Hq, Hkv, Sq, Sk, D, window, sinks = 2, 4, 2, 200, 3000, 128, 2000, 4  # sixteen query tiles of eight CTAs
    q, k, v, _ = make_inputs(B, Hq, Hkv, Sq, Sk, D, torch.bfloat16, seed=8)
    at = torch.tensor([2500, 20], dtype=torch.int32, device="cuda")
    q.requires_grad_()
    with torch.no_grad():
        api().sliding_window_attention(q, k, v, window=window, sinks=sinks, query_start=at)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = api().sliding_window_attention(q, k, v, window=window, sinks=sinks, query_start=at)
        for positions in ([2500, 20], [0, 2800], [-500, 1400]):
            at.copy_(torch.tensor(positions, dtype=torch.int32))
            graph.replay()
            want = api().sliding_window_attention(q, k, v, window=window, sinks=sinks, query_start=at)
            assert torch.equal(out, want)
            mask = window_mask(positions, Sq, Sk, window, sinks)
            exact = ao.math_reference([t.detach().cpu() for t in (q, k, v)], q.detach().cpu(), mask, False, None)[0]
            for b in range(B):
                if mask[b].any():
                    assert ao.per_head_relative_error(out[b:b + 1].cpu(), exact[b:b + 1]) < TOL[torch.bfloat16]["norm"]
    assert native().device_status(reset=True) == 0


@pytest.mark.parametrize("Sq", (1, 300))
def test_captured_calls_follow_new_positions(Sq):
    B, Hq, Hkv, Sk, D, window, sinks = 3, 8, 2, 800, 128, 200, 4
    q, k, v, _ = make_inputs(B, Hq, Hkv, Sq, Sk, D, torch.bfloat16, seed=7)
    at = torch.tensor([400, 20, 0], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        api().sliding_window_attention(q, k, v, window=window, sinks=sinks, query_start=at)
        graphs, outs = [], []
        for _ in range(2):  # two graphs alive at once, replayed in turn
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(api().sliding_window_attention(q, k, v, window=window, sinks=sinks, query_start=at))
            graphs.append(graph)
        for positions in ([400, 20, 0], [499, 300, 77], [-5, 700, 250]):
            at.copy_(torch.tensor(positions, dtype=torch.int32))
            want = api().sliding_window_attention(q, k, v, window=window, sinks=sinks, query_start=at)
            for graph, out in zip(graphs, outs):
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want)


def test_training_step_in_a_graph_and_on_another_stream():
    q, k, v, dout = make_inputs(1, 4, 2, 500, 500, 128, torch.bfloat16, seed=3)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def step():
        out = api().sliding_window_attention(*leaves, window=150, sinks=4)
        return (out, *torch.autograd.grad(out, leaves, dout))

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.detach().clone() for t in step()]
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [t.detach() for t in step()]
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, held))


@pytest.mark.parametrize("D", (64, 128))
def test_repeated_calls_are_bit_identical(D):
    q, k, v, dout = make_inputs(1, 4, 2, 1536, 1536, D, torch.bfloat16, seed=6)
    first = None
    for _ in range(25):
        got = run_attention(api().sliding_window_attention, q, k, v, dout, window=300, sinks=5)
        assert all(bool(torch.isfinite(t).all()) for t in got)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    assert native().device_status(reset=True) == 0


def test_compiled_route():
    q, k, v, dout = make_inputs(1, 4, 2, 200, 200, 64, torch.bfloat16, seed=5)
    want = run_attention(api().sliding_window_attention, q, k, v, dout, window=50, sinks=2)

    def f(q, k, v):
        return api().sliding_window_attention(q, k, v, window=50, sinks=2)

    got = run_attention(torch.compile(f, fullgraph=True, backend="aot_eager"), q, k, v, dout)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals():
    q, k, v, _ = make_inputs(2, 4, 2, 8, 8, 64, torch.bfloat16, seed=5)
    f = api().sliding_window_attention
    at = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="gradients need one query_start"):
        f(q.clone().requires_grad_(True), k, v, window=4, query_start=at)
    with pytest.raises(ValueError, match="int32"):
        f(q, k, v, window=4, query_start=at.cpu())
    with pytest.raises(ValueError, match="FP16/BF16"):
        f(q.float(), k.float(), v.float(), window=4)
    with pytest.raises(ValueError, match="divisible"):
        f(q[:, :3], k, v, window=4)
    with pytest.raises(ValueError, match="window >= 1"):
        native().window_forward(q, k, v, None, 0, 0, 0, 0.1)
    with pytest.raises(ValueError, match="position >= 0"):
        out, m, l = native().window_forward(q, k, v, None, 0, 4, 0, 0.1)
        native().window_backward(q, k, v, out, m, l, out, -1, 4, 0, 0.1)
    with pytest.raises(ValueError, match="int32"):
        native().window_forward(q, k, v, at[:1], 0, 4, 0, 0.1)
    assert native().device_status(reset=True) == 0


def test_nan_stays_where_a_cluster_shares_the_keys():
    """One CTA per query tile or a cluster of them: what is not a number stays visible in every row that sees it."""
    q, k, v, _ = make_inputs(1, 2, 1, 128, 5000, 128, torch.bfloat16, seed=5)
    q[0, 1, 7, 30] = float("nan")     # a whole row of one head
    k[0, 0, 3000, 5] = float("nan")   # seen by the rows from position 3000 to 4999
    v[0, 0, 4000, 9] = float("inf")   # a channel of the rows that see it
    start, window = 4800, 1900        # rows at 4800 .. 4927, windows from 2901 .. 3028 on
    k_seen = (4800 + torch.arange(128)) - window < 3000
    with torch.no_grad():
        got = api().sliding_window_attention(q, k, v, window=window, sinks=4, query_start=start).cpu()
    leaf = q.clone().requires_grad_(True)
    kept = api().sliding_window_attention(leaf, k, v, window=window, sinks=4, query_start=start).detach().cpu()
    for out in (got, kept):
        assert bool(torch.isnan(out[0, 1, 7]).all())
        assert bool(torch.isnan(out[0, :, k_seen]).all())
        rest = ~k_seen
        rest[7] = False
        assert bool((~torch.isfinite(out[0, :, rest][..., 9])).all())
        others = [c for c in range(128) if c != 9]
        assert bool(torch.isfinite(out[0, :, rest][..., others]).all())
    assert native().device_status(reset=True) == 0


def test_compiled_decoding_keeps_no_statistics():
    """A compiled call that nobody differentiates is the eager one: the decoding kernels serve it."""
    q, k, v, _ = make_inputs(3, 8, 2, 1, 600, 128, torch.bfloat16, seed=12)
    at = torch.tensor([599, 3, 250], dtype=torch.int32, device="cuda")

    def f(q, k, v, at):
        return api().sliding_window_attention(q, k, v, window=200, sinks=4, query_start=at)

    def decoded():
        return native().launch_stats().get("window_decode", 0)

    compiled = torch.compile(f, fullgraph=True, backend="aot_eager")
    want = f(q, k, v, at)
    for grad in (True, False):  # nothing requires a gradient; nothing is recorded
        with torch.set_grad_enabled(grad):
            before = decoded()
            got = compiled(q if grad else q.clone().requires_grad_(True), k, v, at)
            assert decoded() > before
            assert torch.equal(got, want) and got.stride() == want.stride()
    narrow = [t[..., :80] for t in make_inputs(2, 4, 2, 70, 300, 96, torch.float16, seed=13)[:3]]  # the tensor-memory forward

    def g(q, k, v):
        return api().sliding_window_attention(q, k, v, window=100, query_start=20, scale=0.2)

    a, b = g(*narrow), torch.compile(g, fullgraph=True, backend="aot_eager")(*narrow)
    assert torch.equal(a, b) and a.stride() == b.stride()


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("Sk", (400, 30000))  # one cluster; a line of blocks cut over all CTAs
def test_decoding_with_a_large_common_score(Sk, dtype):
    """Scores of about 2^20 that differ by a few units, small integers throughout, so that every score is exact: warps and
    CTAs have references of their own, and their parts are weighted alike.  Blocks of 16 keys, which the warps take in
    turn, hold values that tell them apart."""
    D, Hq = 64, 4
    gen = torch.Generator().manual_seed(Sk)
    k = torch.randint(-2, 3, (1, 1, Sk, D), generator=gen).double()
    q = torch.randint(-1, 2, (1, Hq, 1, D), generator=gen).double()
    q[..., 8:] = 0
    q[..., 0], k[..., 0] = 512, 2048
    v = torch.randint(-1, 2, (1, 1, Sk, D), generator=gen).double() / 64 + (torch.arange(Sk) // 16 % 4 + 1).view(1, 1, Sk, 1)
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    with torch.no_grad():
        got = api().sliding_window_attention(q, k, v, window=Sk, query_start=Sk - 1, scale=0.5)
    s = q.cpu().double() @ k.cpu().double().transpose(-1, -2) * 0.5
    prob, vd = torch.softmax(s, -1), v.cpu().double()
    out, u = prob @ vd, 1.1 * torch.finfo(dtype).eps / 2
    # the output's rounding and that of the probabilities; FP32 steps, on differences of scores, in the tenth
    assert bool(((got.cpu().double() - out).abs() <= u * out.abs() + u * (prob @ vd.abs())).all())
    assert native().device_status(reset=True) == 0


def test_dense_rows_off_a_16_byte_boundary_run_on_the_same_kernels():
    """A contiguous view that starts at an odd element: the same results, and no launch of the CUDA-core kernels."""
    def shifted(x):
        return torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)

    def step(tensors):
        leaves = [t.detach().requires_grad_(True) for t in tensors[:3]]
        out = api().sliding_window_attention(*leaves, window=90, sinks=3)
        return out.detach(), *torch.autograd.grad(out, leaves, tensors[3])

    aligned = make_inputs(1, 4, 2, 300, 300, 64, torch.float16, seed=15)
    want = step(aligned)
    before = native().launch_stats()
    for which in (0, 1, 2, 3):
        got = step([shifted(t) if i == which else t for i, t in enumerate(aligned)])
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    with torch.no_grad():
        q, k, v = (t[:, :, -1:].contiguous() if i == 0 else t for i, t in enumerate(aligned[:3]))
        call = dict(window=90, query_start=299)
        one = api().sliding_window_attention(q, k, v, **call)
        for operands in ((shifted(q), k, v), (q, shifted(k), v), (q, k, shifted(v))):
            assert torch.equal(one, api().sliding_window_attention(*operands, **call))
    after = native().launch_stats()
    assert all(after[name] == before.get(name, 0) for name in after if name.startswith("general"))


def test_windows_and_sinks_of_any_size():
    """Integers of any size: beyond 64 bits they are as long as the sequence, not what is left of them in 64 bits."""
    q, k, v, dout = make_inputs(1, 4, 2, 130, 200, 64, torch.bfloat16, seed=14)
    f = api().sliding_window_attention
    for window, sinks, same in ((2**64 + 5, 0, dict(window=1000, sinks=0)), (5, 2**64, dict(window=5, sinks=200)),
                                (2**63, 2**70 + 3, dict(window=1000, sinks=200)), (2**62, 2**62, dict(window=1000, sinks=200))):
        call = dict(window=window, sinks=sinks)
        want = run_attention(f, q, k, v, dout, query_start=60, **same)
        assert all(torch.equal(a, b) for a, b in zip(want, run_attention(f, q, k, v, dout, query_start=60, **call)))
        compiled = torch.compile(lambda q, k, v: f(q, k, v, query_start=60, **call), fullgraph=True, backend="aot_eager")
        with torch.no_grad():
            assert torch.equal(compiled(q, k, v), f(q, k, v, query_start=60, **same))
        cache = api().quantized_cache(1, 2, 200, 64)
        api().quantized_cache_write(cache, k, v)
        few = q[:, :, :2]
        assert torch.equal(api().quantized_cache_attention(few, cache, query_start=150, **call),
                           api().quantized_cache_attention(few, cache, query_start=150, **same))
