"""The compiled host path of the window and cache calls: the same results as the Python one, and its errors."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


def api():
    import kohakufa_cute

    return kohakufa_cute


def native():
    from kohakufa_cute import native

    return native


def rows(*shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


@pytest.fixture
def counted(monkeypatch):
    """The module with its served calls counted; the first call of a process binds the library and is Python's."""
    if native().fast is None:
        pytest.skip("the optional module is not built")
    warm = rows(1, 1, 1, 64)
    api().sliding_window_attention(warm, warm, warm, window=1)

    class Counted:
        served = 0

        def __getattr__(self, name):
            def call(*arguments):
                result = getattr(fast, name)(*arguments)
                self.served += result is not None
                return result

            return call

    fast, module = native().fast, Counted()
    monkeypatch.setattr(native(), "fast", module)
    return module


def without(monkeypatch, call):
    with monkeypatch.context() as patch:
        patch.setattr(native(), "fast", None)
        return call()


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("shape", (
    # B, Hq, Hkv, Sq, Sk, D, window, sinks, start, scale
    (2, 4, 2, 300, 300, 64, 70, 3, 0, None),
    (1, 4, 1, 200, 500, 128, 1000, 0, 100, -0.3),    # the cache is longer than what the queries see
    (1, 2, 2, 130, 130, 96, 1, 0, 0, 0.0),
    (1, 2, 1, 70, 70, 256, 30, 2, 0, None),
    (2, 2, 2, 64, 64, 40, 5, 100, 0, 0.5),
))
def test_training_is_the_same_both_ways(shape, dtype, counted, monkeypatch):
    B, Hq, Hkv, Sq, Sk, D, window, sinks, start, scale = shape
    q, k, v = rows(B, Hq, Sq, D, dtype=dtype, seed=1), rows(B, Hkv, Sk, D, dtype=dtype, seed=2), rows(B, Hkv, Sk, D, dtype=dtype, seed=3)
    dout = rows(B, Hq, Sq, D, dtype=dtype, seed=4)

    def step(leaves, dout):
        leaves = [t.detach().requires_grad_(grad) for t, grad in zip(leaves, (True, True, False))]
        out = api().sliding_window_attention(*leaves, window=window, sinks=sinks, query_start=start, scale=scale)
        return [out.detach(), *torch.autograd.grad(out, leaves[:2], dout)]

    strided = [torch.cat([t, t], -1).transpose(1, 2).contiguous().transpose(1, 2)[..., :D] for t in (q, k, v)]
    shared = [q, k[:1].expand_as(k), v[:1].expand_as(v)]
    for operands, gradient, served in (((q, k, v), dout, 1), (strided, dout[:, :, :1].expand_as(dout), 1),
                                       (shared, dout, int(B == 1))):
        before = counted.served
        got = step(operands, gradient)
        assert counted.served - before == served
        want = without(monkeypatch, lambda: step(operands, gradient))
        for a, b in zip(got, want):
            assert a.stride() == b.stride() and torch.equal(a, b)
    assert native().device_status(reset=True) == 0


def test_serving_is_the_same_both_ways(counted, monkeypatch):
    B, Hq, Hkv, n, D = 3, 8, 2, 200, 128
    k, v, q = rows(B, Hkv, n, D, seed=5), rows(B, Hkv, n, D, seed=6), rows(B, Hq, 2, D, seed=7)
    at = torch.tensor([100, 0, 40], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([7, 200, 0], dtype=torch.int32, device="cuda")

    def step():
        cache = api().quantized_cache(B, Hkv, 300, D)
        api().quantized_cache_write(cache, k, v, start=at, lengths=lengths)
        api().quantized_cache_write(cache, k[:, :, :1], v[:, :, :1], start=299)
        with torch.no_grad():
            return [*cache, *api().quantized_cache_read(cache), *api().quantized_cache_read(cache, start=at, length=9),
                    *api().quantized_cache_read(cache, start=290),
                    api().quantized_cache_attention(q, cache, query_start=at),
                    api().quantized_cache_attention(q, cache, query_start=298, window=50, sinks=2, scale=-0.1),
                    api().sliding_window_attention(q, k, v, window=50, sinks=2, query_start=at),
                    api().sliding_window_attention(q, k, v, window=50, query_start=20, scale=0.2)]

    got = step()
    assert counted.served == 9
    for a, b in zip(got, without(monkeypatch, step)):
        assert torch.equal(a, b) and a.stride() == b.stride()


def test_what_python_serves(counted):
    """Anything that needs more than the launch, or is wrong, is left to the Python layer."""
    fast = counted
    q, cache = rows(1, 2, 3, 64), api().quantized_cache(1, 2, 8, 64)
    window = (4, 0, 0, None)
    misaligned = rows(1, 2, 3, 72)[..., 4:68]
    for call in (lambda: fast.window_attention(q, q, q), lambda: fast.window_attention(q, q, q, True, 0, 0, None),
                 lambda: fast.window_attention(q, q, q, 4, 0, 0, 1), lambda: fast.window_attention(q, q, q, 2**70, 0, 0, None),
                 lambda: fast.window_attention(q, q, q, 4, 0, -1, None), lambda: fast.window_attention(q, q, q, 4, 0, 0, float("nan")),
                 lambda: fast.window_attention(q.cpu(), q, q, *window), lambda: fast.window_attention(q, q[:, :, :2], q, *window),
                 lambda: fast.window_attention(q, misaligned, q, *window), lambda: fast.window_attention(q.float(), q, q, *window),
                 lambda: fast.window_attention(q[..., :7], q[..., :7], q[..., :7], *window),
                 lambda: fast.window_attention(torch.nn.Buffer(q), None, q, *window),
                 lambda: fast.window_attention(q[:, :, :0], q, q, *window),
                 lambda: fast.cache_write(cache, q, q, 6, None), lambda: fast.cache_write(cache[:3], q, q, 0, None),
                 lambda: fast.cache_write(cache, q.half(), q.half(), 0, None), lambda: fast.cache_write(cache, q, q, 0, 3),
                 lambda: fast.cache_write(cache, q.clone().requires_grad_(), q, 0, None),
                 lambda: fast.cache_read(cache, 8, None), lambda: fast.cache_read(cache, 0, 9), lambda: fast.cache_read(cache, 0, True),
                 lambda: fast.cache_attention(q, cache, 0, None, 1, None), lambda: fast.cache_attention(q, cache, 0, 0, 0, None),
                 lambda: fast.cache_attention(q.clone().requires_grad_(), cache, 0, None, 0, None)):
        assert call() is None
    assert not any(t.any() for t in cache)


def test_graph_node_behaves(counted):
    """Saved tensors are version-checked and released, hooks and checkpointing see them, the graph can be kept."""
    q, k, v = (rows(1, 2, 100, 64, seed=s).requires_grad_() for s in (1, 2, 3))
    call = dict(window=20, sinks=1)
    out = api().sliding_window_attention(q, k, v, **call)
    out.sum().backward(retain_graph=True)
    first = [t.grad.clone() for t in (q, k, v)]
    assert all(float(t.abs().sum()) > 0 for t in first[2:])
    out.sum().backward()
    assert all(torch.equal(t.grad, 2 * g) for t, g in zip((q, k, v), first))
    with pytest.raises(RuntimeError, match="second time"):
        out.sum().backward()
    out = api().sliding_window_attention(q, k, v, **call)
    with torch.no_grad():
        k.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or t.cpu(), lambda t: t.cuda()):
        out = api().sliding_window_attention(q, k, v, **call)
    assert len(packed) == 6
    grads = torch.autograd.grad(out.sum(), (q, k, v))
    again = checkpoint(lambda *t: api().sliding_window_attention(*t, **call), q, k, v, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(again.sum(), (q, k, v))))
    with torch.no_grad():  # (other kernels than under a graph: nobody asks for the row statistics)
        plain = api().sliding_window_attention(q, k, v, **call)
    with torch.inference_mode():
        assert torch.equal(api().sliding_window_attention(q, k, v, **call), plain)


def test_second_derivatives_are_refused_both_ways(counted, monkeypatch):
    q, k, v = (rows(1, 2, 100, 64, seed=s).requires_grad_() for s in (1, 2, 3))

    def twice():
        out = api().sliding_window_attention(q, k, v, window=9)
        grad, = torch.autograd.grad(out.sum(), q, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            (grad.float().square().sum() + q.float().sum()).backward()
        return grad.detach()

    out = api().sliding_window_attention(q, k, v, window=9)
    want, = torch.autograd.grad(out.sum(), q)
    assert torch.equal(twice(), want) and torch.equal(without(monkeypatch, twice), want)


def test_a_report_of_a_wait_that_ran_out_reaches_both_directions(counted):
    q = rows(1, 2, 200, 64).requires_grad_()
    out = api().sliding_window_attention(q, q, q, window=20)
    try:
        native().self_test_wait(2_000_000, 1)  # about a millisecond
        torch.cuda.synchronize()
        with pytest.raises(native().DeviceTimeoutError):
            api().sliding_window_attention(q, q, q, window=20)
        with pytest.raises(native().DeviceTimeoutError):
            out.sum().backward()
    finally:
        native().device_status(reset=True)
    torch.autograd.grad(api().sliding_window_attention(q, q, q, window=20).sum(), q)
    assert native().device_status() == 0


def test_forward_mode_is_refused_both_ways(counted, monkeypatch):
    """A tangent would be dropped: an error instead, also where nothing requires a gradient."""
    forward_ad = torch.autograd.forward_ad
    q, k, v = (rows(1, 2, 100, 64, seed=s) for s in (1, 2, 3))
    cache = api().quantized_cache(1, 2, 100, 64)
    calls = (lambda q, k, v: api().sliding_window_attention(q, k, v, window=9),
             lambda q, k, v: api().quantized_cache_write(cache, k, v),
             lambda q, k, v: api().quantized_cache_attention(q[:, :, :2], cache, query_start=98))

    def dual():
        with forward_ad.dual_level():
            for n, call in enumerate(calls):
                for which in ((0, 1, 2), (1, 2), (0,))[n]:
                    operands = [q, k, v]
                    operands[which] = forward_ad.make_dual(operands[which], torch.ones_like(q))
                    with pytest.raises(ValueError, match="forward-mode"):
                        call(*operands)
                    operands[which] = forward_ad.make_dual(operands[which].detach().requires_grad_(), torch.ones_like(q))
                    with pytest.raises(ValueError, match="forward-mode|gradients"):
                        call(*operands)
                call(q, k, v)  # (without a tangent)
        with pytest.raises(ValueError, match="forward-mode"):
            torch.func.jvp(lambda q: calls[0](q, k, v), (q,), (torch.ones_like(q),))

    dual()
    without(monkeypatch, dual)


def test_writes_count_as_changes_in_place(counted, monkeypatch):
    """A cache tensor that autograd has saved is known to have changed, as after any in-place operation of torch."""
    k = rows(1, 2, 3, 64)

    def write():
        cache = api().quantized_cache(1, 2, 8, 64)
        before = [t._version for t in cache]
        x = torch.ones_like(cache.v_params, requires_grad=True)
        product = (x * cache.v_params).sum()  # saves the values
        api().quantized_cache_write(cache, k, k)
        assert all(t._version > n for t, n in zip(cache, before))
        with pytest.raises(RuntimeError, match="inplace"):
            product.backward()
        view = api().QuantizedCache(*(t[:, :, 4:] for t in cache))
        before = [t._version for t in cache]
        api().quantized_cache_write(view, k, k)
        assert all(t._version > n for t, n in zip(cache, before))
        with torch.inference_mode():  # (tensors that keep no count)
            held = api().quantized_cache(1, 2, 8, 64)
            api().quantized_cache_write(held, k, k)
        assert torch.equal(held.k_codes[:, :, :3], cache.k_codes[:, :, :3])

    served = counted.served
    write()
    assert counted.served == served + 3
    without(monkeypatch, write)
