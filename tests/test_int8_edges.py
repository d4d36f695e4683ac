"""The 8-bit operators at the edges of what they are documented to take: values that lie on a tie, single rows of odd length,
scales far from one, inputs that carry a tangent, and calls under a tracer or a dispatch mode."""
import pytest
import torch

from tests.test_int8 import DTYPES, U, gen, half_step, randn, rows_int8


def assert_nearest(x, q):
    """``q`` holds the integers nearest to 127 x / a, ties to even, a the row's largest magnitude.  Checked in integers: with
    at most 24 bits in x and a, 254 x and 2 q a have 32 each, and where q is not 0 their exponents differ by at most nine, so
    that float64 holds both and their difference exactly (where q is 0 the difference is 254 x itself)."""
    a = x.double().abs().amax(-1, keepdim=True)
    v = q.values.double()
    off = (254 * x.double() - 2 * v * a).abs()
    assert bool((off <= a).all()), int((off > a).sum())
    tie = (off == a) & (a > 0)
    assert bool((q.values[tie] % 2 == 0).all()), int((q.values[tie] % 2 != 0).sum())
    return int(tie.sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 33, 1000, 4096, 40960])
def test_values_on_a_tie_and_near_one(dim, dtype):
    """Rows whose largest value is each bfloat16 mantissa and which hold half of it (an exact tie at 63.5), rows of multiples
    of a 254th of their largest (every value a tie or an integer) and their neighbours in the type, at sizes over the range."""
    from coda_gqa_l_b200 import quantize_int8
    g = gen(dim)
    rows = []
    for scale in (1.0, 2.0 ** -92, 2.0 ** 116):
        r = randn(g, 128, dim)
        a = torch.arange(128, 256, device="cuda").float()
        r = r / r.abs().amax(1, keepdim=True) * a[:, None] * 0.99
        r[:, 0], r[:, 1], r[:, dim // 2], r[:, -1] = a, a / 2, -a / 2, a / 2
        rows.append(r * scale)
        n = torch.arange(1, 9, device="cuda").float()[:, None]                    # a = 127 n: ties at odd multiples of n / 2
        h = torch.randint(-254, 255, (8, dim), generator=g, device="cuda").float() / 2 * n
        h[:, 0] = 127 * n[:, 0]
        rows.append(h * scale)
    x = torch.cat(rows).to(dtype)
    assert assert_nearest(x, quantize_int8(x)) > 3 * 128 * 3
    if dtype == torch.float32:
        near = torch.cat([x.nextafter(torch.full_like(x, s * 3e38)) for s in (1, -1)])
        near[:, 0] = torch.cat([x[:, 0]] * 2)                                      # (the largest stays the largest)
        near = near.clamp(-near[:, :1], near[:, :1])
        assert_nearest(near, quantize_int8(near))
    r = randn(g, 300, dim, dtype=dtype)
    assert_nearest(r, quantize_int8(r))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_quotient_of_two_8_bit_mantissas(dtype):
    """A row for each mantissa of its largest value, with every mantissa at every exponent that can still round to one or more
    below it and some under that, both signs: all there is among bfloat16 rows, up to powers of two."""
    from coda_gqa_l_b200 import quantize_int8
    m = torch.arange(128, 256, device="cuda").double()
    below = (m[:, None] * torch.tensor([2.0 ** -i for i in range(14)], device="cuda", dtype=torch.float64)).reshape(-1)
    y = torch.cat([below, -below])[None, :].expand(128, -1)
    y = torch.where(y.abs() <= m[:, None], y, torch.zeros_like(y))
    for scale in (1.0, 2.0 ** -92, 2.0 ** 116):
        x = (torch.cat([m[:, None], y], dim=1) * scale).to(dtype)
        assert torch.equal(x.double(), torch.cat([m[:, None], y], dim=1) * scale)
        assert assert_nearest(x, quantize_int8(x)) >= 2 * 128


@pytest.mark.gpu
def test_single_rows_of_odd_length_are_used_in_place():
    """One row has no distance to another: rows of this package's own making are neither copied nor moved, a product allocates
    its result and nothing else, as it does for two rows."""
    from coda_gqa_l_b200 import Int8Rows, int8_linear, quantize_int8
    g = gen(3)
    w = quantize_int8(randn(g, 40, 577))

    def blocks(call):
        call()
        torch.cuda.synchronize()
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        out = call()
        return torch.cuda.memory_stats()["allocation.all.allocated"] - before, out

    for shape in ((1, 577), (1, 1, 577), (577,), (2, 577)):
        q = quantize_int8(randn(g, *shape))
        n, y = blocks(lambda: int8_linear(q, w, dtype=torch.float32))
        assert n == 1, shape
        ref = (q.values.double() * q.scale.double()[..., None]) @ (w.values.double() * w.scale.double()[:, None]).t()
        mag = (q.values.double().abs() * q.scale.double()[..., None]) @ (w.values.double().abs() * w.scale.double()[:, None]).t()
        assert bool(((y.double() - ref).abs() <= 6 * U * mag).all())
        n, d = blocks(lambda: q.dequantize(torch.float32))
        assert n == 1 and torch.equal(d, q.values.float() * q.scale[..., None])
    # one weight row, and a single row that does not start on a 16-byte boundary (copied)
    q, one = quantize_int8(randn(g, 3, 577)), quantize_int8(randn(g, 1, 577))
    n, y = blocks(lambda: int8_linear(q, one, dtype=torch.float32))
    assert n == 1 and y.shape == (3, 1)
    buf = torch.zeros(600, device="cuda", dtype=torch.int8)
    off = buf[3:580].view(1, 577).copy_(one.values)
    assert torch.equal(int8_linear(q, Int8Rows(off, one.scale), dtype=torch.float32), y)
    assert torch.equal(Int8Rows(off, one.scale).dequantize(torch.float32), one.dequantize(torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(3, 64, 40), (40, 100, 300), (300, 64, 300)])
def test_scales_whose_product_leaves_the_range(m, k, n, dtype):
    """A token's scale far below one with a channel's scale below it, and both far above: the product of the two is not a normal
    number although the result is; and a sum of zero stays zero.  Three roundings as everywhere: u each."""
    from coda_gqa_l_b200 import Int8Rows, int8_linear
    g = gen(m)
    xv, xs = rows_int8(g, m, k)
    wv, ws = rows_int8(g, n, k)
    for sx, sw in ((2.0 ** -98, 2.0 ** -30), (2.0 ** -30, 2.0 ** -98), (2.0 ** -98, 2.0 ** -36)):
        a, b = Int8Rows(xv, (1 + xs * 50) * sx), Int8Rows(wv, (1 + ws * 50) * sw)
        y = int8_linear(a, b, dtype=dtype)
        ref = (xv.double() @ wv.double().t()) * a.scale.double()[:, None] * b.scale.double()
        err = (y.double() - ref).abs()
        normal = ref.abs() > 2.0 ** -125
        assert int(normal.sum()) > m * n // 2
        assert bool((err <= ref.abs() * (4 * U + half_step(dtype)))[normal].all())
        assert bool((err <= 2.0 ** -133)[~normal].all())
    zero = torch.zeros_like(xv)
    y = int8_linear(Int8Rows(zero, torch.full_like(xs, 2.0 ** 100)), Int8Rows(wv, torch.full_like(ws, 2.0 ** 60)), dtype=dtype)
    assert not bool(y.any()) and not bool(y.isnan().any())


def calls_with(t):
    """Every call that takes an activation, with ``t`` applied to that activation; the first one also takes weights."""
    from coda_gqa_l_b200 import Int8Rows, add_rms_norm, int8_linear, quantize_int8
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    q, p = quantize_int8(x), quantize_int8(torch.randn(8, 64, device="cuda"))
    res = torch.zeros(4, 8, device="cuda")
    return (lambda: quantize_int8(t(x)), lambda: add_rms_norm(t(x), w), lambda: add_rms_norm(t(x), w, int8=True),
            lambda: add_rms_norm(x, w, residual=t(x)), lambda: Int8Rows(q.values, t(q.scale)).dequantize(),
            lambda: int8_linear(Int8Rows(q.values, t(q.scale)), p), lambda: int8_linear(q, p, residual=t(res), dtype=torch.float32))


@pytest.mark.gpu
def test_inputs_with_a_tangent_are_refused():
    """The tangent of a dual number, an activation's or a weight's, is refused and not dropped."""
    import torch.autograd.forward_ad as fa

    from coda_gqa_l_b200 import Int8Rows, add_rms_norm, int8_linear, quantize_int8
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    q, p = quantize_int8(x), quantize_int8(torch.randn(8, 64, device="cuda"))
    b = torch.zeros(8, device="cuda")
    with fa.dual_level():
        dual = lambda t: fa.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (*calls_with(dual), lambda: add_rms_norm(x, dual(w)), lambda: int8_linear(q, Int8Rows(p.values, dual(p.scale))),
                     lambda: int8_linear(q, p, dual(b), dtype=torch.float32)):
            with pytest.raises(RuntimeError, match="inference"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="inference"):
                call()
        for call in calls_with(lambda t: t):
            call()


@pytest.mark.gpu
def test_activations_that_need_a_gradient_are_refused():
    """The scales of 8-bit activations among them, and a parameter too where activations are meant; weights may be parameters."""
    from coda_gqa_l_b200 import Int8Rows, add_rms_norm, int8_linear, quantize_int8
    for call in (*calls_with(lambda t: t.clone().requires_grad_()), *calls_with(torch.nn.Parameter)[1:]):
        with pytest.raises(RuntimeError, match="inference"):
            call()
        with torch.no_grad():
            call()
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    q, p = quantize_int8(torch.nn.Parameter(x)), quantize_int8(torch.randn(8, 64, device="cuda"))
    add_rms_norm(x, torch.nn.Parameter(w))
    int8_linear(q, Int8Rows(p.values, torch.nn.Parameter(p.scale)), torch.nn.Parameter(torch.zeros(8, device="cuda")), dtype=torch.float32)


def test_gradients_are_refused_under_a_dispatch_mode_too():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from coda_gqa_l_b200 import Int8Rows, add_rms_norm, int8_linear, quantize_int8
    with FakeTensorMode():
        x, w = torch.empty(4, 64, device="cuda"), torch.ones(64, device="cuda")
        q, p = quantize_int8(x), quantize_int8(torch.empty(8, 64, device="cuda"))
        g = torch.empty(4, 64, device="cuda", requires_grad=True)
        res = torch.empty(4, 8, device="cuda", requires_grad=True)
        scale = torch.empty(4, device="cuda", requires_grad=True)
        for call in (lambda: quantize_int8(g), lambda: add_rms_norm(g, w), lambda: add_rms_norm(g, w, int8=True),
                     lambda: add_rms_norm(x, w, residual=g), lambda: Int8Rows(q.values, scale).dequantize(),
                     lambda: int8_linear(Int8Rows(q.values, scale), p), lambda: int8_linear(q, p, residual=res, dtype=torch.float32)):
            with pytest.raises(RuntimeError, match="inference"):
                call()
            with torch.no_grad():
                call()
        quantize_int8(torch.nn.Parameter(x))
        add_rms_norm(x, torch.nn.Parameter(w))


@pytest.mark.gpu
def test_a_traced_call_follows_its_inputs():
    """torch.jit.trace records the operators, not the values they had."""
    from coda_gqa_l_b200 import add_rms_norm, int8_linear, quantize_int8
    g = gen(9)
    w, nw = quantize_int8(randn(g, 24, 64)), 1 + 0.1 * randn(g, 64)

    def f(x, r):
        q, h = add_rms_norm(x, nw, residual=r, int8=True)
        return int8_linear(q, w, dtype=torch.float32), h, quantize_int8(x).dequantize(torch.float32), add_rms_norm(r, nw)[0]

    a, b = [(randn(g, 5, 64), randn(g, 5, 64)) for _ in range(2)]
    with torch.no_grad():
        traced = torch.jit.trace(f, a, check_trace=False)
        for args in (a, b):
            assert all(torch.equal(p, q) for p, q in zip(traced(*args), f(*args)))


@pytest.mark.gpu
def test_rows_written_and_read_back_to_back_through_the_same_memory():
    """Each call reads what the one before it on the stream has just written where the call before that one wrote something
    else: scales and values never come from an earlier round."""
    from coda_gqa_l_b200 import quantize_int8
    g = gen(17)
    for rows, dim, dtype in ((1, 64, torch.float32), (40, 1000, torch.bfloat16), (300, 512, torch.bfloat16), (2000, 4096, torch.bfloat16)):
        xs = [randn(g, rows, dim, dtype=dtype) * 4.0 ** i for i in range(5)]
        want = [quantize_int8(x).dequantize(dtype).clone() for x in xs]
        torch.cuda.synchronize()
        bad = torch.zeros((), device="cuda", dtype=torch.int64)
        for i in range(200):
            q = quantize_int8(xs[i % 5])
            bad += (q.dequantize(dtype) != want[i % 5]).sum()
            del q
        assert int(bad) == 0


def test_c_entries_refuse_addresses_between_two_elements():
    """What a kernel would read or write with accesses of an element's size starts on one's boundary, or the call is refused on
    the host (a misaligned access would end the context)."""
    from coda_gqa_l_b200._lib import lib
    ok, odd, two = 4096, 4097, 4098                                # never read: every call is refused on the host

    def refused(rc):
        assert rc == -1 and b"boundar" in lib.coda_b200_last_error(), (rc, lib.coda_b200_last_error())

    for dtype, bad in ((1, odd), (0, two), (0, odd)):
        names = ("x", "r", "w", "sum", "y")
        for name in names:
            a = dict.fromkeys(names, ok) | {name: bad}
            refused(lib.coda_b200_add_rms_norm(dtype, 4, 8, a["x"], 8, a["r"], 8, a["w"], 1e-6, a["sum"], 8, a["y"], 8, None, 0, None, None))
        refused(lib.coda_b200_quantize_rows(dtype, 4, 8, bad, 8, ok, 16, ok, None))
        refused(lib.coda_b200_dequantize_rows(dtype, 4, 8, ok, 16, ok, bad, 8, None))
        for name in ("b", "r", "y"):
            a = dict(b=ok, r=ok, y=ok) | {name: bad}
            refused(lib.coda_b200_int8_gemm(dtype, 4, 64, 8, ok, 64, ok, ok, 64, ok, a["b"], a["r"], 8, a["y"], 8, 0, None, None))
    refused(lib.coda_b200_add_rms_norm(1, 4, 8, ok, 8, None, 0, ok, 1e-6, None, 0, None, 0, ok, 16, two, None))
    refused(lib.coda_b200_quantize_rows(1, 4, 8, ok, 8, ok, 16, two, None))
    refused(lib.coda_b200_dequantize_rows(1, 4, 8, ok, 16, two, ok, 8, None))
    for scales in ((two, ok), (ok, two)):
        refused(lib.coda_b200_int8_gemm(1, 4, 64, 8, ok, 64, scales[0], ok, 64, scales[1], None, None, 0, ok, 8, 0, None, None))
    refused(lib.coda_b200_int8_gemm(1, 4, 64, 8, ok, 64, ok, ok, 64, ok, None, None, 0, ok, 8, 0, two, None))


@pytest.mark.gpu
def test_a_wait_of_the_product_that_runs_out_reports_and_releases_the_cta():
    """The bounded wait of the 8-bit product on barriers nobody arrives at: the short one gives up and leaves its code in the
    status word and the CTA's abort word, the long one of the same CTA leaves on seeing that; the context stays usable."""
    from coda_gqa_l_b200._lib import check, lib
    s = torch.cuda.current_stream().cuda_stream
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    report = torch.full((5,), -1, dtype=torch.int32, device="cuda")
    check(lib.coda_b200_selftest_int8_wait(2048, status.data_ptr(), report.data_ptr(), s), "coda_b200_selftest_int8_wait")
    torch.cuda.synchronize()
    r = report.tolist()
    assert int(status) == 48 and r[0] == 0 and r[2] == 0 and r[4] == 48, r
    assert r[3] <= 4 * r[1] + 100_000, r                       # (released by the abort word, not by its own limit 2048 times as long)
    assert float((torch.ones(8, device="cuda") * 2).sum()) == 16.0
    for limit, st, rep in ((0, status, report), (65537, status, report)):
        with pytest.raises(RuntimeError):
            check(lib.coda_b200_selftest_int8_wait(limit, st.data_ptr(), rep.data_ptr(), None), "coda_b200_selftest_int8_wait")


@pytest.mark.gpu
def test_a_call_that_waits_for_room_in_the_queue_lets_other_threads_run():
    """More launches than the queue of a busy stream holds: while they wait, other Python threads go on (one may hold what the
    stream is waiting for)."""
    import threading
    import time

    from coda_gqa_l_b200 import add_rms_norm, int8_linear, quantize_int8
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    p = quantize_int8(torch.randn(8, 64, device="cuda"))
    gap, stop = [0.0], threading.Event()

    def tick():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gap[0], last = max(gap[0], now - last), now

    q = quantize_int8(x)
    int8_linear(q, p), q.dequantize(), add_rms_norm(x, w)
    for call in (lambda: quantize_int8(x), lambda: q.dequantize(), lambda: add_rms_norm(x, w), lambda: int8_linear(q, p)):
        torch.cuda.synchronize()
        gap[0] = 0.0
        stop.clear()
        thread = threading.Thread(target=tick)
        thread.start()
        torch.cuda._sleep(1_200_000_000)                        # some 0.6 s
        t0 = time.perf_counter()
        for _ in range(3000):
            call()
        waited = time.perf_counter() - t0
        stop.set()
        thread.join()
        assert waited > 0.3 and gap[0] < 0.2, (waited, gap[0])
    torch.cuda.synchronize()
