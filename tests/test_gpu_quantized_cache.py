"""The 4-bit key/value cache: written bits against the definition, what stays untouched, reading back, and attention
to it against FP64 mathematics on the values it holds."""

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = (torch.bfloat16, torch.float16)


def api():
    import kohakufa_cute

    return kohakufa_cute


def native():
    from kohakufa_cute import native as module

    return module


def rows(*shape, dtype, seed, offset=True):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    if offset:
        x = x + 2 * torch.randn((1, shape[1], 1, shape[3]), generator=gen)
    return x.to(dtype).cuda()


def quantise(x):
    """The definition, on the CPU in IEEE FP32: (codes as bytes, params) of x [..., D]."""
    g = x.cpu().float().unflatten(-1, (-1, 64))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((high - low) / 15).to(x.dtype)
    step = scale.float()
    code = torch.where(step > 0, torch.round((g - low) / torch.where(step > 0, step, 1.0)), 0.0).clamp(0, 15)
    code = code.flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat((scale, low.to(x.dtype)), -1)


def values(codes, params):
    """FP64 values of a cache half."""
    codes, params = codes.cpu(), params.cpu().double()
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double().unflatten(-1, (-1, 64))
    return (params[..., 1:2] + params[..., 0:1] * code).flatten(-2)


def filled(B, H, capacity, D, dtype, seed):
    """A cache whose every row holds something, and clones of its tensors."""
    cache = api().quantized_cache(B, H, capacity, D, dtype=dtype)
    api().quantized_cache_write(cache, rows(B, H, capacity, D, dtype=dtype, seed=seed),
                                rows(B, H, capacity, D, dtype=dtype, seed=seed + 1, offset=False))
    return cache


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ((1, 1, 1, 64), (2, 3, 37, 128), (1, 2, 5, 256), (2, 1, 300, 512), (3, 2, 129, 64)))
def test_written_bits_equal_the_definition(shape, dtype):
    B, H, n, D = shape
    k, v = rows(*shape, dtype=dtype, seed=n), rows(*shape, dtype=dtype, seed=n + 1, offset=False)
    k[0, 0, 0, :64] = 3.0  # a group of equal values
    v[0, 0, 0, :64] = 0.0
    v[0, 0, 0, 5] = torch.finfo(dtype).tiny / 4  # the scale underflows, or nearly
    cache = api().quantized_cache(B, H, n + 3, D, dtype=dtype)
    api().quantized_cache_write(cache, k, v, start=2)
    for x, codes, params in ((k, cache.k_codes, cache.k_params), (v, cache.v_codes, cache.v_params)):
        want_codes, want_params = quantise(x)
        assert torch.equal(codes[:, :, 2:n + 2].cpu(), want_codes)
        assert torch.equal(params[:, :, 2:n + 2].cpu(), want_params)
        for t in (codes, params):
            assert not t[:, :, :2].any() and not t[:, :, n + 2:].any()
    got = api().quantized_cache_read(cache, start=2, length=n)
    for x, half, params in ((k, got[0], cache.k_params), (v, got[1], cache.v_params)):
        want = values(*quantise(x))
        u = torch.finfo(dtype).eps / 2
        # reading rounds once; the product and the sum before it are one FP32 fused multiply-add
        assert bool(((half.cpu().double() - want).abs() <= (u + 2**-22) * want.abs() + torch.finfo(dtype).tiny).all())
        # a code is at most half a step from its value; the rounded scale adds 15 times its own rounding, at the top
        # of the group, and a scale below the normal range is rounded in absolute steps
        scale = params[:, :, 2:n + 2, :, :1].cpu().double().expand(*params.shape[:2], n, D // 64, 64).flatten(-2)
        slack = scale * 0.5 + 15 * (u * scale + torch.finfo(dtype).tiny * torch.finfo(dtype).eps)
        assert bool(((x.cpu().double() - want).abs() <= slack + 2**-22 * x.cpu().double().abs()).all())
    assert native().device_status(reset=True) == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_ragged_rows_leave_the_rest_as_it_was(dtype):
    B, H, n, D, capacity = 5, 2, 33, 128, 100
    cache = filled(B, H, capacity, D, dtype, seed=3)
    before = [t.clone() for t in cache]
    k, v = rows(B, H, n, D, dtype=dtype, seed=8), rows(B, H, n, D, dtype=dtype, seed=9)
    starts, lengths = [0, 67, 90, -10, 2**31 - 5], [33, 20, 33, 33, 0]
    at = torch.tensor(starts, dtype=torch.int32, device="cuda")
    many = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    api().quantized_cache_write(cache, k, v, start=at, lengths=many)
    want = [t.cpu().clone() for t in before]
    for x, codes, params in ((k, want[0], want[1]), (v, want[2], want[3])):
        new_codes, new_params = quantise(x)
        for b in range(B):
            for r in range(lengths[b]):
                if 0 <= starts[b] + r < capacity:
                    codes[b, :, starts[b] + r], params[b, :, starts[b] + r] = new_codes[b, :, r], new_params[b, :, r]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(cache, want))
    got = api().quantized_cache_read(cache, start=at, length=n)
    for half, codes, params in ((got[0], want[0], want[1]), (got[1], want[2], want[3])):
        whole = values(codes, params).to(dtype)
        for b in range(B):
            for r in range(n):
                inside = 0 <= starts[b] + r < capacity
                row = half[b, :, r].cpu()
                if inside:
                    torch.testing.assert_close(row, whole[b, :, starts[b] + r], atol=0, rtol=torch.finfo(dtype).eps)
                else:
                    assert not row.any()
    long = torch.full((B,), 1000, dtype=torch.int32, device="cuda")  # longer than the rows given: all of them
    api().quantized_cache_write(cache, k, v, start=0, lengths=long)
    assert torch.equal(cache.k_codes[:, :, :n].cpu(), quantise(k)[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_written_bits_over_the_range_of_the_type(dtype):
    """Groups of every magnitude the type has, wide and narrow, with many quotients at or next to a half: the bits equal
    IEEE FP32 arithmetic."""
    gen = torch.Generator().manual_seed(77)
    n, D = 4096, 256
    low, high = (-14, 14) if dtype == torch.float16 else (-120, 120)
    power = torch.randint(low, high, (1, 1, n, D // 64, 1), generator=gen).double()
    x = torch.randn(1, 1, n, D // 64, 64, generator=gen).double() * torch.exp2(power)
    steps = torch.randint(0, 31, (1, 1, n, D // 64, 64), generator=gen).double() * 0.5 * torch.exp2(power)  # multiples of a half
    x = torch.where(torch.arange(n).view(1, 1, n, 1, 1) % 2 == 0, x, steps)
    x = torch.where(torch.arange(n).view(1, 1, n, 1, 1) % 5 == 0, x * torch.exp2(-8.0 * torch.rand(x.shape, generator=gen)), x)
    x = x.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype).flatten(-2).cuda()
    cache = api().quantized_cache(1, 1, n, D, dtype=dtype)
    api().quantized_cache_write(cache, x, x.flip(-1))
    for half, codes, params in ((x, cache.k_codes, cache.k_params), (x.flip(-1), cache.v_codes, cache.v_params)):
        want_codes, want_params = quantise(half)
        finite = torch.isfinite(want_params[..., 0].float())
        assert torch.equal(params.cpu()[..., 0][finite], want_params[..., 0][finite])
        rows_codes = codes.cpu().unflatten(-1, (-1, 32))
        assert torch.equal(rows_codes[finite], want_codes.unflatten(-1, (-1, 32))[finite])


def test_values_that_are_not_finite():
    for dtype in TYPES:
        k = rows(1, 1, 4, 128, dtype=dtype, seed=1)
        k[0, 0, 0, 3], k[0, 0, 1, 70], k[0, 0, 2, 127] = float("nan"), float("inf"), -float("inf")
        v = torch.full_like(k, torch.finfo(dtype).max)
        v[..., ::2] = -torch.finfo(dtype).max
        cache = api().quantized_cache(1, 1, 4, 128, dtype=dtype)
        api().quantized_cache_write(cache, k, v)
        got, wide = api().quantized_cache_read(cache)
        want = values(*quantise(k)).to(dtype)
        for r, group in ((0, 0), (1, 1), (2, 1)):
            assert bool(torch.isnan(got[0, 0, r, group * 64:(group + 1) * 64]).all())
            other = slice((1 - group) * 64, (2 - group) * 64)
            torch.testing.assert_close(got[0, 0, r, other].cpu(), want[0, 0, r, other], atol=0, rtol=torch.finfo(dtype).eps)
        if dtype == torch.float16:  # the widest range of FP16 is held
            assert bool(torch.isfinite(wide).all()) and float((wide.float() - v.float()).abs().max()) <= 65504 * 2**-9
        else:  # a range beyond FP32 is not
            assert bool(torch.isnan(wide).all())


def test_layouts_of_rows_and_cache():
    B, H, n, D = 2, 4, 50, 128
    k, v = rows(B, H, n, D, dtype=torch.bfloat16, seed=4), rows(B, H, n, D, dtype=torch.bfloat16, seed=5)
    plain = api().quantized_cache(B, H, 64, D)
    api().quantized_cache_write(plain, k, v, start=7)
    seen = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]  # [B, n, H, D] in memory
    odd = torch.zeros(B, H, n, D + 1, device="cuda", dtype=torch.bfloat16)
    odd[..., 1:] = v
    big = api().quantized_cache(B + 1, H + 2, 80, D)
    view = type(big)(*(t[1:, 1:H + 1, 8:72] for t in big))
    api().quantized_cache_write(view, seen[0], odd[..., 1:], start=7)
    for a, b in zip(plain, view):
        assert torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(api().quantized_cache_read(plain), api().quantized_cache_read(view)))
    assert not big.k_codes[0].any() and not big.k_codes[:, 0].any() and not big.k_codes[:, :, 72:].any()
    q = rows(B, 2 * H, 1, D, dtype=torch.bfloat16, seed=6)
    want = api().quantized_cache_attention(q, plain, query_start=50)
    assert torch.equal(want, api().quantized_cache_attention(q, view, query_start=50))
    spread = torch.zeros(B, 2 * H, 1, 2 * D, device="cuda", dtype=torch.bfloat16)
    spread[..., ::2] = q
    assert torch.equal(want, api().quantized_cache_attention(spread[..., ::2], view, query_start=50))


def reference(q, cache, starts, window, sinks, scale=None):
    """(out, bound) in FP64.  The bound: the output's rounding, and the probabilities' (each enters the product
    multiplied by its key's scale and rounded, against codes less 8) - u |O| + u sum_c P 8 scale_c; FP32 steps (score
    sums, ex2, normaliser) below 3e-5 of sum_c P |V| are covered by a tenth of u of it."""
    B, Hq, Sq, D = q.shape
    k, v = values(cache.k_codes, cache.k_params), values(cache.v_codes, cache.v_params)
    steps = cache.v_params[..., 0].cpu().double().repeat_interleave(64, -1)
    group, Sk = Hq // k.shape[1], k.shape[2]
    pos = torch.tensor(starts)[:, None, None] + torch.arange(Sq)[None, :, None]
    key = torch.arange(Sk)[None, None]
    seen = key <= pos
    if window:
        seen = seen & ((key > pos - window) | (key < sinks))
    seen = seen[:, None]
    k, v, steps = (t.nan_to_num(0.0, 0.0, 0.0).repeat_interleave(group, 1) for t in (k, v, steps))
    s = q.cpu().double() @ k.transpose(-1, -2) * (D**-0.5 if scale is None else scale)
    blind = ~seen.any(-1, keepdim=True)
    s = s.masked_fill(~seen, float("-inf")).masked_fill(blind, 0.0)
    p = torch.softmax(s, -1).masked_fill(~seen, 0.0)
    u = torch.finfo(q.dtype).eps / 2
    out = p @ v
    bound = u * out.abs() + u * 8 * (p @ steps) + 0.1 * u * (p @ v.abs()) + torch.finfo(q.dtype).tiny
    return out, bound


CASES = (
    # Hq, Hkv, Sq, capacity, D, window, sinks, starts
    (8, 8, 1, 1, 64, 0, 0, (0,)),
    (8, 8, 1, 777, 64, 0, 0, (776,)),
    (32, 8, 1, 2000, 128, 0, 0, (1999, 0, 31, 32, 1000)),
    (8, 1, 4, 1500, 128, 0, 0, (1496, 5, -2, 2**31 - 1)),     # 32 rows per cache head, rows before the first key
    (6, 2, 3, 900, 128, 100, 4, (897, 99, 0, 950)),           # nine rows; behind the cache: sinks and a part of the window
    (16, 2, 1, 3000, 64, 256, 130, (2999, 385, 200)),
    (4, 4, 2, 700, 128, 33, 0, (698, 64, 800)),               # the last sequence sees nothing
    (5, 1, 7, 513, 64, 1, 1, (506, 0)),
    (64, 8, 4, 1100, 128, 4096, 4, (1096, 512)),
    (2, 1, 40, 400, 128, 64, 16, (360, 17)),                  # a longer piece
    (8, 2, 1, 300, 128, 0, 0, tuple(range(0, 280, 4))),       # seventy sequences
    (12, 1, 1, 5000, 64, 700, 3, (4999, 2500)),               # twelve rows per cache head
    (4, 1, 1, 40000, 128, 0, 0, (39999,)),                    # one long sequence over many CTAs
)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_attention_matches_fp64(case, dtype):
    Hq, Hkv, Sq, capacity, D, window, sinks, starts = case
    B = len(starts)
    cache = filled(B, Hkv, capacity, D, dtype, seed=capacity)
    q = rows(B, Hq, Sq, D, dtype=dtype, seed=capacity + 7, offset=False) * 1.5
    for b, start in enumerate(starts):  # behind the last position there may be anything
        end = min(capacity, max(0, start + Sq))
        for codes, params in (cache[:2], cache[2:]):
            codes[b, :, end:], params[b, :, end:] = 255, float("nan")
    at = torch.tensor(starts, dtype=torch.int32, device="cuda")
    for scale in (None, -0.2):
        want, bound = reference(q, cache, starts, window, sinks, scale)
        got = api().quantized_cache_attention(q, cache, query_start=at, window=window or None, sinks=sinks, scale=scale)
        assert got.shape == q.shape and got.dtype == dtype and bool(torch.isfinite(got).all())
        far = ((got.cpu().double() - want).abs() - bound).max()
        assert float(far) <= 0, f"an element is {float(far):.3e} beyond its roundings"
        again = api().quantized_cache_attention(q, cache, query_start=at, window=window or None, sinks=sinks, scale=scale)
        assert torch.equal(got, again)
    if 0 <= starts[0] < 2**31 - 1:
        one = type(cache)(*(t[:1] for t in cache))
        same = api().quantized_cache_attention(q[:1], one, query_start=starts[0], window=window or None, sinks=sinks,
                                               scale=-0.2)
        want, bound = reference(q[:1], one, starts[:1], window, sinks, -0.2)
        assert bool(((same.cpu().double() - want).abs() <= bound).all())
    assert native().device_status(reset=True) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", (
    # both sides of the rule that chooses between one cluster per unit and a line of blocks cut over all CTAs, and
    # clusters of every size:  Hq, Hkv, Sq, capacity, D, window, sinks, starts
    (4, 4, 1, 96 * 64, 128, 0, 0, (96 * 64 - 1, -1, 500)),         # the longest that clusters take, and the next
    (4, 4, 1, 96 * 64 + 1, 128, 0, 0, (96 * 64, -1, 500)),
    (16, 8, 1, 333, 128, 0, 0, tuple(range(-2, 333, 61))),         # 48 units: eight CTAs each
    (16, 8, 1, 333, 128, 0, 0, tuple(range(-2, 333, 49))),         # 56: seven
    (16, 8, 1, 333, 128, 0, 0, tuple(range(-2, 333, 43))),         # 64: six
    (16, 8, 1, 700, 128, 0, 0, tuple(range(-2, 700, 79))),         # 72: five
    (16, 8, 1, 700, 128, 200, 3, tuple(range(-2, 700, 54))),       # 104: three
    (16, 8, 1, 600, 128, 0, 0, tuple(range(-2, 600, 33))),         # 152: two
    (16, 8, 1, 400, 128, 0, 0, tuple(range(-2, 400, 11))),         # 296: one
    (16, 8, 1, 200, 128, 0, 0, tuple(range(-2, 200, 4))),          # 408: the line
    (32, 2, 4, 700, 64, 150, 9, tuple(range(-6, 720, 53))),        # 32 rows, two units per cache head
    (12, 1, 1, 900, 128, 0, 0, tuple(range(-1, 900, 23))),         # 40 units of 16 rows
    (12, 1, 1, 300, 128, 0, 0, tuple(range(-1, 300, 1))),          # 301: the line
))
def test_short_and_full_batches(case, dtype):
    Hq, Hkv, Sq, capacity, D, window, sinks, starts = case
    cache = filled(len(starts), Hkv, capacity, D, dtype, seed=capacity + 3)
    q = rows(len(starts), Hq, Sq, D, dtype=dtype, seed=capacity + 11, offset=False) * 1.5
    at = torch.tensor(starts, dtype=torch.int32, device="cuda")
    want, bound = reference(q, cache, starts, window, sinks)
    got = api().quantized_cache_attention(q, cache, query_start=at, window=window or None, sinks=sinks)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    assert native().device_status(reset=True) == 0


def test_a_zero_scale_averages_the_visible_values():
    cache = filled(1, 2, 300, 128, torch.bfloat16, seed=5)
    q = rows(1, 4, 1, 128, dtype=torch.bfloat16, seed=6)
    want, bound = reference(q, cache, (200,), 40, 3, 0.0)
    got = api().quantized_cache_attention(q, cache, query_start=200, window=40, sinks=3, scale=0.0)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


def test_launches_are_counted():
    cache = filled(1, 2, 9000, 128, torch.bfloat16, seed=3)
    q = rows(1, 8, 1, 128, dtype=torch.bfloat16, seed=4)
    for window, launches in ((100, 1), (None, 2)):  # one cluster per K/V head; a line of blocks and its merge
        before = native().launch_count()
        api().quantized_cache_attention(q, cache, query_start=8999, window=window)
        assert native().launch_count() - before == launches


def test_large_logits_pick_one_key():
    """Scores that differ by hundreds: the softmax is a copy of one value row."""
    for dtype in TYPES:
        cache = filled(1, 1, 2000, 128, dtype, seed=11)
        q = (rows(1, 8, 1, 128, dtype=dtype, seed=12) * 100).to(dtype)
        want, bound = reference(q, cache, (1999,), 0, 0)
        got = api().quantized_cache_attention(q, cache, query_start=1999)
        # FP32 score sums of magnitude up to 100 * 128 * 10 are off by 2^-22 of that: 0.03, a factor 1.03 in P where a
        # second key comes close (bounded by the values' own size), nothing where it does not
        slack = 0.03 * values(cache.v_codes, cache.v_params).abs().max()
        assert bool(((got.cpu().double() - want).abs() <= bound + slack).all())


def test_captured_decoding_follows_new_positions():
    """Write one token, attend, in a graph; replayed with other rows and positions it equals eager calls."""
    B, Hq, Hkv, D, capacity = 3, 8, 2, 128, 1200
    eager, held = filled(B, Hkv, capacity, D, torch.bfloat16, 1), filled(B, Hkv, capacity, D, torch.bfloat16, 1)
    k, v = rows(B, Hkv, 1, D, dtype=torch.bfloat16, seed=2), rows(B, Hkv, 1, D, dtype=torch.bfloat16, seed=3)
    q = rows(B, Hq, 1, D, dtype=torch.bfloat16, seed=4)
    at = torch.tensor([700, 3, 0], dtype=torch.int32, device="cuda")

    def step(cache, window):
        api().quantized_cache_write(cache, k, v, start=at)
        return api().quantized_cache_attention(q, cache, query_start=at, window=window, sinks=4 if window else 0)

    graphs = []
    for window in (None, 300):
        step(held, window)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(held, window)
        graphs.append((graph, out, window))
    step(eager, None)
    for i, positions in enumerate(([701, 4, 1], [1199, 600, 0], [20, 1198, 333])):
        at.copy_(torch.tensor(positions, dtype=torch.int32))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(t.dtype))
        for graph, out, window in graphs:
            want = step(eager, window)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(eager, held))


def test_another_stream_and_two_calls_at_once():
    cache = filled(2, 2, 4000, 128, torch.bfloat16, 21)
    q = rows(2, 8, 1, 128, dtype=torch.bfloat16, seed=22)
    want = api().quantized_cache_attention(q, cache, query_start=3999)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(10):
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append(api().quantized_cache_attention(q, cache, query_start=3999))
    torch.cuda.synchronize()
    assert all(torch.equal(want, r) for r in results)


def test_decoding_steps_follow_a_prompt():
    """A prompt written and attended to, then tokens one by one: each step equals attention on what was read back."""
    B, Hq, Hkv, D, prompt, steps, window, sinks = 2, 8, 2, 128, 300, 4, 128, 4
    cache = api().quantized_cache(B, Hkv, prompt + steps, D)
    k, v = (rows(B, Hkv, prompt + steps, D, dtype=torch.bfloat16, seed=s) for s in (31, 32))
    q = rows(B, Hq, prompt + steps, D, dtype=torch.bfloat16, seed=33)
    api().quantized_cache_write(cache, k[:, :, :prompt], v[:, :, :prompt])
    kq, vq = api().quantized_cache_read(cache, length=prompt)
    out = api().sliding_window_attention(q[:, :, :prompt], kq, vq, window=window, sinks=sinks)
    want, bound = reference(q[:, :, :prompt], type(cache)(*(t[:, :, :prompt] for t in cache)), (0, 0), window, sinks)
    # the window operator reads K and V rounded to 16 bits, which the direct definition does not: one more rounding of
    # V (u sum P |V|), and scores off by u sum |q| |k| / sqrt(D), i.e. P off by that factor
    u = torch.finfo(torch.bfloat16).eps / 2
    kd, vd = (t.cpu().double().repeat_interleave(Hq // Hkv, 1) for t in (kq, vq))
    factor = u * (q[:, :, :prompt].cpu().double().abs() @ kd.abs().transpose(-1, -2)).amax(-1, keepdim=True) * D**-0.5
    slack = (2 * u + 2 * factor) * vd.abs().amax(2, keepdim=True)
    assert bool(((out.cpu().double() - want).abs() <= bound + slack).all())
    for t in range(prompt, prompt + steps):
        api().quantized_cache_write(cache, k[:, :, t:t + 1], v[:, :, t:t + 1], start=t)
        got = api().quantized_cache_attention(q[:, :, t:t + 1], cache, query_start=t, window=window, sinks=sinks)
        want, bound = reference(q[:, :, t:t + 1], cache, (t, t), window, sinks)
        assert bool(((got.cpu().double() - want).abs() <= bound).all())
    assert native().device_status(reset=True) == 0


def test_offsets_past_32_bits():
    """A cache whose planes are longer than 4 GiB: rows near the end are written, read and attended to in place."""
    capacity, D = (1 << 26) + 4096, 128  # 64 bytes of codes per token and plane
    codes = [torch.empty((1, 2, capacity, D // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    params = [torch.empty((1, 2, capacity, D // 64, 2), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache = api().QuantizedCache(codes[0], params[0], codes[1], params[1])
    n, start = 200, capacity - 203
    k, v = rows(1, 2, n, D, dtype=torch.bfloat16, seed=51), rows(1, 2, n, D, dtype=torch.bfloat16, seed=52)
    q = rows(1, 4, 1, D, dtype=torch.bfloat16, seed=53)
    api().quantized_cache_write(cache, k, v, start=start)
    small = api().quantized_cache(1, 2, n, D)
    api().quantized_cache_write(small, k, v)
    far, near = (api().quantized_cache_read(c, start=s, length=n) for c, s in ((cache, start), (small, 0)))
    assert all(torch.equal(a, b) for a, b in zip(far, near))
    got = api().quantized_cache_attention(q, cache, query_start=start + n - 1, window=n)
    want, bound = reference(q, small, (n - 1,), n, 0)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


def test_a_cache_that_overlaps_itself_is_read_but_not_written():
    cache = filled(1, 2, 64, 64, torch.bfloat16, 61)
    shared = api().QuantizedCache(*(t.expand(3, *t.shape[1:]) for t in cache))  # one prefix for three sequences
    q = rows(3, 4, 1, 64, dtype=torch.bfloat16, seed=62)
    got = api().quantized_cache_attention(q, shared, query_start=63)
    for b in range(3):
        assert torch.equal(got[b:b + 1], api().quantized_cache_attention(q[b:b + 1], cache, query_start=63))
    k = rows(3, 2, 1, 64, dtype=torch.bfloat16, seed=63)
    with pytest.raises(ValueError, match="overlap"):
        api().quantized_cache_write(shared, k, k)


def test_compiled_route():
    cache, other = (filled(2, 2, 200, 64, torch.float16, 41) for _ in range(2))
    k, v = rows(2, 2, 3, 64, dtype=torch.float16, seed=42), rows(2, 2, 3, 64, dtype=torch.float16, seed=43)
    q = rows(2, 4, 3, 64, dtype=torch.float16, seed=44)

    def step(q, k, v, cache):
        api().quantized_cache_write(cache, k, v, start=100)
        out = api().quantized_cache_attention(q, cache, query_start=100, window=50, sinks=2)
        return out, *api().quantized_cache_read(cache, start=90, length=13)

    want = step(q, k, v, cache)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, v, other)
    assert all(torch.equal(a, b) for a, b in zip((*want, *cache), (*got, *other)))


def test_refusals():
    cache = api().quantized_cache(2, 2, 16, 64)
    k = rows(2, 2, 4, 64, dtype=torch.bfloat16, seed=1)
    q = rows(2, 4, 1, 64, dtype=torch.bfloat16, seed=1)
    write, read, attend = api().quantized_cache_write, api().quantized_cache_read, api().quantized_cache_attention
    for call in (lambda: write(cache, k, k, start=13), lambda: write(cache, k, k[:, :, :3]),
                 lambda: write(cache, k.half(), k.half()), lambda: write(cache, k[:1], k[:1]),
                 lambda: write(cache, k.cpu(), k.cpu()), lambda: write(cache, k, k, lengths=4),
                 lambda: write(cache, k.clone().requires_grad_(True), k),
                 lambda: read(cache, start=10, length=7), lambda: read(cache, length=0), lambda: read(cache, start=16),
                 lambda: read(cache, start=torch.zeros(2, dtype=torch.int32, device="cuda")),
                 lambda: attend(q[:, :3], cache, query_start=0), lambda: attend(q.half(), cache, query_start=0),
                 lambda: attend(q, cache, query_start=0, sinks=2), lambda: attend(q, cache, query_start=0, window=0),
                 lambda: attend(q.clone().requires_grad_(True), cache, query_start=0),
                 lambda: attend(q, cache, query_start=0, scale=float("inf")),
                 lambda: attend(q, cache, query_start=torch.zeros(2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: native().cache_write(k, k, *cache, None, None, 2**31), lambda: native().cache_read(*cache, None, -2**40, 1),
                 lambda: native().cache_attention(q, *cache, None, 2**62, 0, 0, 0.1)):
        with pytest.raises(ValueError, match="32 bits"):  # (the public calls refuse these before the library does)
            call()
    wide = api().quantized_cache(1, 1, 4, 256)
    with pytest.raises(ValueError, match="64 and 128"):
        attend(rows(1, 1, 1, 256, dtype=torch.bfloat16, seed=1), wide, query_start=0)
    shifted = torch.zeros(2 * 2 * 16 * 32 + 8, dtype=torch.uint8, device="cuda")[8:].view(2, 2, 16, 32)
    with pytest.raises(ValueError, match="aligned"):
        write(cache._replace(k_codes=shifted), k, k)
    assert all(not t.any() for t in cache)
    assert native().device_status(reset=True) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", (192, 320, 384, 448, 128))
def test_params_may_start_at_any_pair(D, dtype):
    """Rows of any number of groups, wherever the allocator puts the params: their bases at successive multiples of 512
    bytes, as torch allocates, and in between.  Written bits and what is read back equal the definition."""
    B, H, n, capacity = 2, 2, 21, 30
    k, v = rows(B, H, n, D, dtype=dtype, seed=D), rows(B, H, n, D, dtype=dtype, seed=D + 1, offset=False)
    shape, size = (B, H, capacity, D // 64, 2), B * H * capacity * (D // 64) * 2
    want = [quantise(x) for x in (k, v)]
    wide = [torch.zeros(B, H, capacity, D // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for at in (0, 256, 512, 768, 1024, 1280, 1536, 2, 6, 1030):  # 16-bit elements
        store = [torch.zeros(size + 2048, dtype=dtype, device="cuda") for _ in range(2)]
        assert all(t.data_ptr() % 512 == 0 for t in store)
        params = [t[at + 2 * i:at + 2 * i + size].view(shape) for i, t in enumerate(store)]
        cache = api().QuantizedCache(wide[0], params[0], wide[1], params[1])
        api().quantized_cache_write(cache, k, v, start=4)
        got = api().quantized_cache_read(cache, start=4, length=n)
        for (want_codes, want_params), codes, held, half in zip(want, wide, params, got):
            assert torch.equal(codes[:, :, 4:n + 4].cpu(), want_codes) and torch.equal(held[:, :, 4:n + 4].cpu(), want_params)
            u, exact = torch.finfo(dtype).eps / 2, values(want_codes, want_params)
            assert bool(((half.cpu().double() - exact).abs() <= (u + 2**-22) * exact.abs() + torch.finfo(dtype).tiny).all())
        for i, t in enumerate(store):  # nothing around them was written
            assert not t[:at + 2 * i].any() and not t[at + 2 * i + size:].any()
    assert native().device_status(reset=True) == 0


def test_attention_wants_a_tokens_params_in_one_piece():
    """Attention copies a token's scales and zeros at once: 8 bytes at 128 channels, 4 at 64."""
    for D, at, served in ((64, 2, True), (128, 4, True), (128, 2, False)):
        B, H, capacity = 1, 2, 40
        shape, size = (B, H, capacity, D // 64, 2), B * H * capacity * (D // 64) * 2
        plain = filled(B, H, capacity, D, torch.bfloat16, seed=D)
        moved = []
        for held in (plain.k_params, plain.v_params):
            store = torch.zeros(size + 64, dtype=torch.bfloat16, device="cuda")[at:at + size].view(shape)
            moved.append(store.copy_(held))
        cache = plain._replace(k_params=moved[0], v_params=moved[1])
        assert all(torch.equal(a, b) for a, b in zip(api().quantized_cache_read(plain), api().quantized_cache_read(cache)))
        q = rows(B, 4, 1, D, dtype=torch.bfloat16, seed=3)
        if served:
            want = api().quantized_cache_attention(q, plain, query_start=39)
            assert torch.equal(want, api().quantized_cache_attention(q, cache, query_start=39))
        else:
            with pytest.raises(ValueError, match="aligned"):
                api().quantized_cache_attention(q, cache, query_start=39)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("capacity", (1000, 40000))  # one cluster; a line of blocks cut over all CTAs
def test_a_large_common_score(capacity, dtype):
    """Scores of about 2^20 that differ by a few units, integers throughout, so that every score is exact: warps and CTAs
    have references of their own, and their parts are weighted alike.  Blocks of 64 tokens hold values that tell them
    apart."""
    gen = torch.Generator().manual_seed(capacity)
    codes = [torch.randint(0, 256, (1, 1, capacity, 64), generator=gen).to(torch.uint8) for _ in range(2)]
    params = [torch.ones(1, 1, capacity, 2, 2) for _ in range(2)]
    codes[0][..., :32] = 0                      # keys: the first group is 256 throughout, the second 0 .. 15
    params[0][..., 0, 1], params[0][..., 1, 1] = 256, 0
    params[1][..., 0] = 2.0**-8                 # values: about 1, 2, 3, 4 by block
    params[1][..., 1] = (torch.arange(capacity) // 64 % 4 + 1).view(1, 1, capacity, 1)
    q = torch.zeros(1, 4, 1, 128)
    q[..., :64] = 64
    q[..., 64:70] = torch.randint(-1, 2, (1, 4, 1, 6), generator=gen)
    cache = api().QuantizedCache(codes[0].cuda(), params[0].to(dtype).cuda(), codes[1].cuda(), params[1].to(dtype).cuda())
    q = q.to(dtype).cuda()
    want, bound = reference(q, cache, (capacity - 1,), 0, 0, 0.5)
    got = api().quantized_cache_attention(q, cache, query_start=capacity - 1, scale=0.5)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    assert native().device_status(reset=True) == 0


def test_the_output_is_laid_out_like_the_queries():
    """Also where the rows cannot be addressed as they are; the compiled route declares the same layout."""
    B, Hq, Sq, D = 2, 4, 3, 64
    cache = filled(B, 2, 200, D, torch.float16, seed=71)
    odd = torch.zeros(B * Sq * Hq * D + 1, dtype=torch.float16, device="cuda")[1:].view(B, Sq, Hq, D).transpose(1, 2)
    odd.copy_(rows(B, Hq, Sq, D, dtype=torch.float16, seed=72))

    def f(q, cache):
        out = api().quantized_cache_attention(q, cache, query_start=100, window=50, sinks=2)
        return out, out.transpose(1, 2).view(B, Sq, Hq * D)

    want = api().quantized_cache_attention(odd.contiguous(), cache, query_start=100, window=50, sinks=2)
    for call in (f, torch.compile(f, fullgraph=True, backend="aot_eager")):
        out, flat = call(odd, cache)
        assert out.stride() == torch.empty_like(odd).stride() and torch.equal(out, want)
        assert torch.equal(flat, want.transpose(1, 2).reshape(B, Sq, Hq * D))


def test_dense_rows_off_a_16_byte_boundary_are_taken():
    """A contiguous view that starts at an odd element: nothing but its address differs."""
    def shifted(x):
        return torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)

    k, v, q = (rows(2, H, 20, 64, dtype=torch.bfloat16, seed=s) for s, H in ((81, 2), (82, 2), (83, 4)))
    cache, other = (api().quantized_cache(2, 2, 30, 64) for _ in range(2))
    api().quantized_cache_write(cache, k, v, start=3)
    api().quantized_cache_write(other, shifted(k), shifted(v), start=3)
    assert all(torch.equal(a, b) for a, b in zip(cache, other))
    few = q[:, :, :2].contiguous()
    want = api().quantized_cache_attention(few, cache, query_start=20)
    assert torch.equal(want, api().quantized_cache_attention(shifted(few), cache, query_start=20))


def test_caches_whose_rows_share_memory_are_not_written():
    """An overlap by any strides, and keys that are the values' own memory, are refused; a stride of an axis of one
    element says nothing."""
    k = rows(2, 2, 5, 64, dtype=torch.bfloat16, seed=64)
    plain = api().quantized_cache(2, 2, 40, 64)
    store = torch.zeros(2 * 2 * 40 * 32, dtype=torch.uint8, device="cuda")
    sliding = store.as_strided((2, 2, 40, 32), (32 * 40, 32 * 20, 32, 1))  # the second head starts inside the first
    pairs = torch.zeros(2 * 2 * 40 * 2, dtype=torch.bfloat16, device="cuda")
    behind = pairs.as_strided((2, 2, 40, 1, 2), (160, 80, 0, 2, 1))        # every token the same pair
    for bad in (plain._replace(k_codes=sliding), plain._replace(v_codes=sliding), plain._replace(k_params=behind),
                plain._replace(v_codes=plain.k_codes), plain._replace(v_params=plain.k_params)):
        with pytest.raises(ValueError, match="overlap"):
            api().quantized_cache_write(bad, k, k)
    assert not store.any() and not pairs.any() and not any(t.any() for t in plain)
    one = api().quantized_cache(1, 2, 40, 64)
    loose = api().QuantizedCache(*(t.as_strided(t.shape, (0, *t.stride()[1:])) for t in one))
    api().quantized_cache_write(loose, k[:1], k[:1], start=3)
    want = api().quantized_cache(1, 2, 40, 64)
    api().quantized_cache_write(want, k[:1], k[:1], start=3)
    assert all(torch.equal(a, b) for a, b in zip(one, want))
    swapped = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in plain]  # [B, capacity, H, ...] in memory
    api().quantized_cache_write(api().QuantizedCache(*swapped), k, k, start=3)
    api().quantized_cache_write(plain, k, k, start=3)
    assert all(torch.equal(a, b) for a, b in zip(swapped, plain))


def test_params_that_require_gradients_are_refused():
    """The calls record nothing, so that a gradient with respect to scales and zeros would be missing without a word."""
    plain = filled(1, 2, 30, 64, torch.bfloat16, seed=65)
    q = rows(1, 2, 1, 64, dtype=torch.bfloat16, seed=66)
    for name in ("k_params", "v_params"):
        cache = plain._replace(**{name: getattr(plain, name).clone().requires_grad_()})
        calls = (lambda: api().quantized_cache_read(cache), lambda: api().quantized_cache_write(cache, q, q),
                 lambda: api().quantized_cache_attention(q, cache, query_start=29))
        for call in calls:
            with pytest.raises(ValueError, match="inference only"):
                call()
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(calls[0](), api().quantized_cache_read(plain)))
            calls[1]()
            assert torch.equal(calls[2](), calls[2]())
