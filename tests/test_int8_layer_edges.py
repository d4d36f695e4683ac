"""Layers and stacks with 8-bit projections on the paths a decoding loop takes (hidden states side by side in memory, with a
residual, without norms), and what has to happen to the layer's derived weight copies when parameters are replaced, when a
first call is captured, and when two streams share a layer."""
import pytest
import torch

from tests.test_int8 import U, check_int8
from tests.test_int8_layer import FIELDS, SHAPES, hidden, layer, piecewise, stack

SMALL = SHAPES[0][1]
BF16 = [s for s in SHAPES if s[0] == torch.bfloat16]


def watch_native(mod):
    """How many eager steps of ``mod`` ran as one native call."""
    taken = [0]
    inner = mod._step_eager_int8

    def spy(x, st, residual):
        y = inner(x, st, residual)
        taken[0] += y is not None
        return y

    mod._step_eager_int8 = spy
    return taken


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kw", BF16)
@pytest.mark.parametrize("bias", [False, True])
def test_native_step_is_its_projections_called_one_by_one(dtype, kw, bias):
    """step(x), step(rows in 8 bits) and step_residual(x) of hidden states as a decoding loop has them, each as one native call:
    the bits of the projections called one by one, the residual added before the result is rounded."""
    from coda_gqa_l_b200 import _deep_copy_state, quantize_int8
    mod = layer(kw, dtype)
    D, B = kw["embed_dim"], 3
    if bias:
        mod.o_proj.bias = torch.nn.Parameter(torch.randn(D, device="cuda").to(dtype))
    ref = piecewise(mod)
    taken = watch_native(mod)
    x = hidden(B, 120, D, dtype, 1)
    torch.manual_seed(2)
    sa = mod.init_state(batch_size=B, device="cuda", dtype=dtype)
    sb = _deep_copy_state(sa)
    for s, m in ((sa, mod), (sb, ref)):
        m.prefill_chunked(x[:, :40], s, block_size=16)
    for t in range(40, 120):
        xt = x[:, t:t + 1].contiguous()
        if t % 3 == 0:
            y, want = mod.step_residual(xt, sa), ref._step_fused(ref._cfg(B, dtype, sb), xt, sb, ring(sb), host_update=True, residual=xt)
        elif t % 3 == 1:
            y, want = mod.step(xt, sa)[0], ref.step(xt, sb)[0]
        else:
            y, want = mod.step(quantize_int8(xt), sa)[0], ref.step(xt, sb)[0]
        assert torch.equal(y, want), t
    assert taken[0] == 80
    for f in FIELDS:
        assert torch.equal(getattr(sa, f), getattr(sb, f)), f
    assert (sa.pos, sa.recent_idx, sa.recent_filled) == (sb.pos, sb.recent_idx, sb.recent_filled) and mod.device_status() == 0


def ring(st):
    from coda_gqa_l_b200._lib import RingPos
    return RingPos(int(st.pos), int(st.recent_idx), int(st.recent_filled), None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kw", SHAPES)
@pytest.mark.parametrize("residual", [True, False])
def test_stack_without_norms_eager_and_captured(dtype, kw, residual):
    """Prefill, eager, captured and host-fed steps of a stack of 8-bit layers without norms against the layers' projections
    called one by one.  (An eager float32 step has no native call: its residual is an addition of its own.)"""
    from coda_gqa_l_b200 import _deep_copy_state
    st = stack(kw, dtype, 3, True, residual, norms=False)
    refs = [piecewise(l) for l in st.layers]
    taken = [watch_native(l) for l in st.layers]
    native = dtype == torch.bfloat16
    B, D = 2, kw["embed_dim"]
    x = hidden(B, 100, D, dtype, 7)
    torch.manual_seed(3)
    s1 = st.init_states(batch_size=B, device="cuda", dtype=dtype)
    s2, s3, s4 = ([_deep_copy_state(s) for s in s1] for _ in range(3))

    def by_hand(h, states, eager):
        for r, s in zip(refs, states):
            if eager and not native:
                h = r.step_residual(h, s) if residual else r.step(h, s)[0]
            else:
                h = r.step_graphable(h, s, ring(s), residual=h if residual else None)
                r.advance_host_scalars(s)
        return h

    a, c = st.prefill(x[:, :70], s1, block_size=24), st.prefill(x[:, :70], s3, block_size=24)
    for states in (s2, s4):
        b = x[:, :70]
        for r, s in zip(refs, states):
            b = r.prefill_chunked_residual(b, s, block_size=24) if residual else r.prefill_chunked(b, s, block_size=24)[0]
        assert torch.equal(a, b) and torch.equal(c, b)
    for t in range(70, 90):
        xt = x[:, t:t + 1].contiguous()
        assert torch.equal(st.step(xt, s1), by_hand(xt, s2, True)), t
        c = st.step_graph(xt, s3) if t % 2 else st.step_graph_host(xt.cpu(), s3)
        torch.cuda.synchronize()
        assert torch.equal(c.cuda(), by_hand(xt, s4, False)), t
    if native:
        assert all(n[0] >= 20 for n in taken)
    for got, want in ((s1, s2), (s3, s4)):
        for f in FIELDS:
            assert all(torch.equal(getattr(p, f), getattr(q, f)) for p, q in zip(got, want)), f
    assert all(l.device_status() == 0 for l in st.layers)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kw", SHAPES)
def test_stack_hands_its_layers_the_norm_in_64_bits(dtype, kw):
    """What each layer of a pre-norm stack is given, against the norm of the residual stream in 64 bits (weight and eps its own)."""
    st = stack(kw, dtype, 3, True)
    for i, n in enumerate(st.norms):
        n.eps = 1e-3 * 10 ** i
    B, D = 2, kw["embed_dim"]
    x = hidden(B, 12, D, dtype, 7)
    torch.manual_seed(3)
    states = st.init_states(batch_size=B, device="cuda", dtype=dtype)
    seen = []

    def spy(call):
        def inner(n, s, **k):
            y, s = call(n, s, **k)
            seen.append((n, y))
            return y, s
        return inner

    for l in st.layers:
        l.prefill_chunked, l.step = spy(l.prefill_chunked), spy(l.step)
    for call, xs in ((lambda v: st.prefill(v, states, block_size=4), x[:, :9]), (lambda v: st.step(v, states), x[:, 9:10])):
        out, h, y = call(xs), xs, None
        for (q, following), norm in zip(seen, st.norms):
            s = h.double() if y is None else h.double() + y.double()              # (not yet rounded to the type)
            check_int8(q, s * torch.rsqrt(s.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.double())
            h, y = (h if y is None else (h.float() + y.float()).to(dtype)), following
        assert len(seen) == 3 and torch.equal(out, h + y)
        seen.clear()


def fresh_like(mod, kw, dtype):
    """A new layer with the parameters that ``mod`` has now."""
    from coda_gqa_l_b200 import CoDAGQALandmarkPerf2
    new = CoDAGQALandmarkPerf2(**kw).eval().to(dtype).cuda()
    if mod.o_proj.bias is not None:
        new.o_proj.bias = torch.nn.Parameter(mod.o_proj.bias.detach().clone())
    new.load_state_dict(mod.state_dict())
    new.use_int8_projections = mod.use_int8_projections
    return new


def new_out(mod):
    n, d, w = mod.num_heads * mod.head_dim, mod.embed_dim, mod.q_proj.weight
    device, dtype = w.device, w.dtype
    del mod.o_proj
    mod.o_proj = torch.nn.Linear(n, d, bias=False, device=device, dtype=dtype)


def set_key(mod):
    mod.k_proj.weight = torch.nn.Parameter(mod.k_proj.weight.detach() * 0.5)


def assigned(mod):
    mod.load_state_dict({k: v * 0.75 if v.is_floating_point() else v.clone() for k, v in mod.state_dict().items()}, assign=True)


def add_bias(mod):
    mod.o_proj.bias = torch.nn.Parameter(torch.ones_like(mod.q_proj.weight[0]))


def no_bias(mod):
    mod.o_proj.bias = None


def swapped(mod):
    """As functional calls do it: past the module's own attribute setting."""
    mod.v_proj._parameters["weight"] = torch.nn.Parameter(mod.v_proj.weight.detach() * -0.5)


CHANGES = (new_out, new_out, set_key, assigned, assigned, swapped, add_bias, no_bias, new_out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kw", SHAPES[:2])
def test_replaced_parameters_reach_the_prefill(dtype, kw):
    """A projection deleted and built anew (its memory may come back at the old address), a parameter set, a state dict assigned
    instead of copied, a bias that comes and goes: the next prefill is that of a fresh layer with the new parameters."""
    from coda_gqa_l_b200 import _deep_copy_state
    mod = layer(kw, dtype)
    x = hidden(2, 30, kw["embed_dim"], dtype, 3)
    torch.manual_seed(2)
    s0 = mod.init_state(batch_size=2, device="cuda", dtype=dtype)
    run = lambda m: m.prefill_chunked(x, _deep_copy_state(s0), block_size=8)[0]  # noqa: E731
    last = run(mod)
    for change in CHANGES:
        with torch.no_grad():
            change(mod)
        got = run(mod)
        assert torch.equal(got, run(fresh_like(mod, kw, dtype))), change.__name__
        assert not torch.equal(got, last), change.__name__
        last = got


def test_copies_know_another_parameter_at_the_same_address(monkeypatch):
    """An output weight that lies where the old one lay and counts as many versions: both kinds of derived copies are made again."""
    mod = on_cpu(monkeypatch)
    with torch.no_grad():
        old_t, old_8 = mod._skinny_weights()[2], mod._int8_weights()[2]
        old = mod.o_proj.weight
        new = torch.nn.Parameter(old.data)
        while new._version < old._version:
            new.mul_(1.0)
        new.detach().numpy()[...] *= -0.5
        mod.o_proj.weight = new
        assert new.data_ptr() == old.data_ptr() and new._version == old._version
        assert torch.equal(mod._skinny_weights()[2], new.t()) and mod._skinny_weights()[2] is not old_t
        now = mod._int8_weights()[2]
        assert now is not old_8 and torch.equal(now.scale, new.abs().amax(1) / 127)
        again = mod._int8_weights()[2]
        assert again is now and mod._skinny_weights() is mod._skinny_weights()       # (and not without a reason)


def on_cpu(monkeypatch=None):
    """A float32 layer on the CPU, for what the host does with its parameters; rows to 8 bits by their formula."""
    from coda_gqa_l_b200 import CoDAGQALandmarkPerf2, Int8Rows, attention
    torch.manual_seed(0)
    mod = CoDAGQALandmarkPerf2(**SMALL).eval()

    def quantise(x):
        scale = x.abs().amax(-1) / 127
        return Int8Rows(torch.round(x / scale[..., None]).to(torch.int8), scale)

    if monkeypatch is not None:
        monkeypatch.setattr(attention, "quantize_int8", quantise)
    return mod


def test_a_capture_leaves_parameters_and_caches_alone(monkeypatch):
    """While a graph is captured nothing has been computed yet: parameters are not moved into memory that the graph fills in its
    replays, no derived copy made then is kept, and the memory that the graph reads the parameters from stays."""
    from coda_gqa_l_b200 import attention
    mod = on_cpu(monkeypatch)
    mod.use_int8_projections = True
    cpu = torch.device("cpu")
    where = {n: p.data_ptr() for n, p in mod.named_parameters()}
    want = torch.cat([l.weight.detach() for l in (mod.q_proj, mod.k_proj, mod.v_proj, mod.lambda_proj, mod.write_proj)])
    monkeypatch.setattr(attention, "_recording", lambda t: True, raising=False)
    with torch.no_grad():
        f = mod._fused_weight()
        assert torch.equal(f[0][:want.shape[0]], want) and not bool(f[0][want.shape[0]:].any())
        assert torch.equal(mod._skinny_weights()[1], f[0].t())
        mod._consts(cpu, torch.float32)
        mod._decode_bundle(cpu, torch.float32)
        mod._int8_weights()
        mod._int8_bundle(cpu, torch.float32)
        assert where == {n: p.data_ptr() for n, p in mod.named_parameters()}
        assert mod._fused is None and mod._wt is None and mod._int8 is None and not mod._const_cache
        assert mod.__dict__.get("_bundle") is None and mod.__dict__.get("_bundle8") is None
        monkeypatch.setattr(attention, "_recording", lambda t: False)
        f = mod._fused_weight()                    # outside: the parameters become rows of one matrix, as ever ...
        assert mod.q_proj.weight.data_ptr() == f[0].data_ptr() != where["q_proj.weight"] and torch.equal(f[0][:want.shape[0]], want)
        kept = {t.data_ptr(): t for t in mod._recorded.values()}               # ... and what the graph reads is still there
        for n in ("q_proj", "k_proj", "v_proj", "lambda_proj", "write_proj"):
            assert torch.equal(kept[where[n + ".weight"]], getattr(mod, n).weight)
            if getattr(mod, n).bias is not None:
                assert torch.equal(kept[where[n + ".bias"]], getattr(mod, n).bias)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [True, False])
def test_first_call_captured_then_replayed_beside_calls_outside(int8):
    """A layer whose first call ever is captured: a call outside before the first replay, replays with the memory around them
    used for other things, a call outside and replays again -- each the result of a layer that was never captured."""
    from coda_gqa_l_b200 import _deep_copy_state
    dtype, kw = SHAPES[1]
    mod, ref = layer(kw, dtype, int8=int8), layer(kw, dtype, int8=int8)
    x = hidden(2, 40, kw["embed_dim"], dtype, 3)
    torch.manual_seed(2)
    s0 = mod.init_state(batch_size=2, device="cuda", dtype=dtype)
    s1 = _deep_copy_state(s0)
    arena = s1._arena.clone()
    run = lambda m, s: m.prefill_chunked(x, s, block_size=16)[0]  # noqa: E731

    def same(a, b):             # (under capture the library may pick another GEMM)
        assert torch.equal(a, b) if int8 else float((a.double() - b.double()).norm() / b.double().norm()) < 2e-2

    want = run(ref, _deep_copy_state(s0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(mod, s1)
    junk = []

    def fill():
        torch.cuda.synchronize()
        for p in list(mod.parameters()):
            junk.extend(torch.full(p.shape, float("nan"), device="cuda", dtype=dtype) for _ in range(3))

    fill()
    assert torch.equal(run(mod, _deep_copy_state(s0)), want)
    for _ in range(3):
        fill()
        s1._arena.copy_(arena)
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        same(got, want)
        assert torch.equal(run(mod, _deep_copy_state(s0)), want)
    assert mod.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [True, False])
def test_replaced_parameters_reach_the_eager_step(int8):
    """The same for the eager step alone, which runs from addresses gathered once."""
    from coda_gqa_l_b200 import _deep_copy_state
    dtype, kw = SHAPES[1]
    mod = layer(kw, dtype, int8=int8)
    x = hidden(2, 4, kw["embed_dim"], dtype, 3)
    torch.manual_seed(2)
    s0 = mod.init_state(batch_size=2, device="cuda", dtype=dtype)

    def run(m):
        s = _deep_copy_state(s0)
        return torch.cat([m.step(x[:, t:t + 1].contiguous(), s)[0] for t in range(4)], dim=1)

    last = run(mod)
    for change in CHANGES:
        with torch.no_grad():
            change(mod)
        got = run(mod)
        assert torch.equal(got, run(fresh_like(mod, kw, dtype))), change.__name__
        assert not torch.equal(got, last), change.__name__
        last = got


@pytest.mark.parametrize("int8", [True, False])
def test_gathered_addresses_know_replaced_parameters(int8, monkeypatch):
    """Each way to replace a parameter makes the eager step gather its addresses again, and nothing else does."""
    mod = on_cpu(monkeypatch)
    mod.use_int8_projections = int8
    gather = lambda: (mod._int8_bundle if int8 else mod._decode_bundle)(torch.device("cpu"), torch.float32)  # noqa: E731
    with torch.no_grad():
        last = gather()
        assert gather() is last
        for change in CHANGES:
            if change is add_bias and not int8:
                break                                  # (gathered without one only)
            change(mod)
            now = gather()
            assert now is not last, change.__name__
            f = mod._fused_weight()
            assert now["layer"].bias == f[1].data_ptr()
            if int8:
                assert now["w8"].out_bias == (None if mod.o_proj.bias is None else mod.o_proj.bias.data_ptr())
                assert now["w8"].w_in == mod._int8_weights()[1].values.data_ptr()
            else:
                assert now["w_in"] == f[0].data_ptr() and now["w_out"] == mod.o_proj.weight.data_ptr()
            assert gather() is now
            last = now
        if not int8:
            add_bias(mod)
            assert gather() is None
            no_bias(mod)
            assert gather() is not None
        mod.rope.inv_freq = mod.rope.inv_freq * 0.5
        now = gather()
        assert now is not last and now["layer"].inv_freq == mod._consts(torch.device("cpu"), torch.float32)[0].data_ptr()


def test_output_bias_of_another_type_takes_the_general_path(monkeypatch):
    """The native step reads the bias in the state's type: it does not take a layer whose output bias has another."""
    mod = on_cpu(monkeypatch)
    mod.use_int8_projections = True
    with torch.no_grad():
        add_bias(mod)
        mod.o_proj.bias = torch.nn.Parameter(mod.o_proj.bias.detach().bfloat16())
        assert mod._int8_bundle(torch.device("cpu"), torch.float32) is None
        mod.o_proj.bias = torch.nn.Parameter(torch.ones(2 * mod.embed_dim)[::2])
        assert mod._int8_bundle(torch.device("cpu"), torch.float32) is None
        add_bias(mod)
        assert mod._int8_bundle(torch.device("cpu"), torch.float32) is not None


def test_copies_are_made_again_into_the_same_memory(monkeypatch):
    """A graph captured around a layer holds the addresses of its 8-bit copies: they stay when the parameters change."""
    from coda_gqa_l_b200 import attention
    mod = on_cpu(monkeypatch)
    with torch.no_grad():
        a = mod._int8_weights()
        where = [t.data_ptr() for r in a[1:3] for t in r]
        for change in (lambda: mod.k_proj.weight.mul_(0.5), lambda: new_out(mod), lambda: assigned(mod),
                       lambda: (mod.o_proj.weight.data.mul_(3.0), mod.refresh_weights())):
            change()
            b = mod._int8_weights()
            assert b is not a and [t.data_ptr() for r in b[1:3] for t in r] == where
            for r, w in ((b[1], mod._fused_weight()[0]), (b[2], mod.o_proj.weight)):
                want = attention.quantize_int8(w.detach())
                assert torch.equal(r.values, want.values) and torch.equal(r.scale, want.scale)
            a = b


@pytest.mark.gpu
def test_two_streams_share_a_layer_that_neither_has_used():
    """The first call of a layer on one stream, held up there, and the second on another with no event between them; then a
    call held up on the second stream while the first changes the weights: each result is that of the weights at its call."""
    from coda_gqa_l_b200 import _deep_copy_state
    dtype, kw = SHAPES[1]
    x = hidden(2, 64, kw["embed_dim"], dtype, 3)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for trial in range(4):
        mod, ref = layer(kw, dtype, seed=trial), layer(kw, dtype, seed=trial)
        torch.manual_seed(trial)
        s0 = mod.init_state(batch_size=2, device="cuda", dtype=dtype)
        states = [_deep_copy_state(s0) for _ in range(6)]
        run = lambda m, s: m.prefill_chunked(x, s, block_size=32)[0]  # noqa: E731
        want = run(ref, states[0])
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            torch.cuda._sleep(4_000_000)                       # some 2 ms
            ya = run(mod, states[1])
        with torch.cuda.stream(b):
            yb = run(mod, states[2])
        torch.cuda.synchronize()
        assert torch.equal(ya, want) and torch.equal(yb, want)
        with torch.cuda.stream(b):
            torch.cuda._sleep(4_000_000)
            yb = run(mod, states[3])
        with torch.cuda.stream(a), torch.no_grad():
            mod.q_proj.weight.mul_(-1.0)
            mod.o_proj.weight.mul_(0.5)
            ya = run(mod, states[4])
        torch.cuda.synchronize()
        assert torch.equal(yb, want)
        with torch.no_grad():
            ref.q_proj.weight.mul_(-1.0)
            ref.o_proj.weight.mul_(0.5)
        assert torch.equal(ya, run(ref, states[5])) and not torch.equal(ya, want)


@pytest.mark.gpu
def test_graph_captured_by_hand_follows_changed_weights():
    """A replay of a graph around a layer's prefill after its weights changed, the old copies' memory having been offered to
    others: the results of the new weights once a call outside has taken them over, of the old ones before."""
    from coda_gqa_l_b200 import _deep_copy_state
    dtype, kw = SHAPES[1]
    mod = layer(kw, dtype)
    x = hidden(2, 40, kw["embed_dim"], dtype, 3)
    torch.manual_seed(2)
    s0 = mod.init_state(batch_size=2, device="cuda", dtype=dtype)
    run = lambda s: mod.prefill_chunked(x, s, block_size=16)[0]  # noqa: E731
    first = run(_deep_copy_state(s0))
    s1 = _deep_copy_state(s0)
    arena = s1._arena.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(s1)

    def replayed():
        s1._arena.copy_(arena)
        graph.replay()
        torch.cuda.synchronize()
        return got.clone()

    assert torch.equal(replayed(), first)
    with torch.no_grad():
        for p in (mod.k_proj.weight, mod.o_proj.weight):
            p.mul_(-0.7)
    assert torch.equal(replayed(), first)
    second = run(_deep_copy_state(s0))
    junk = [torch.full((n,), 77, device="cuda", dtype=torch.int8) for n in (mod._int8[1].values.numel(), mod._int8[2].values.numel()) for _ in range(4)]
    assert torch.equal(replayed(), second) and not torch.equal(second, first)
    mod.refresh_weights()
    junk += [torch.full_like(junk[0], 77) for _ in range(4)]
    assert torch.equal(run(_deep_copy_state(s0)), second) and torch.equal(replayed(), second)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [True, False])
def test_two_streams_and_two_graphs_share_a_layer(int8):
    """Prefills that evict and steps of one layer on two streams side by side, each with states of its own, then two graphs of
    a step replayed side by side: the results of one after the other."""
    from coda_gqa_l_b200 import _deep_copy_state
    dtype, kw = SHAPES[1]
    mod = layer(kw, dtype, int8=int8)
    xs = [hidden(8, 300, kw["embed_dim"], dtype, i) for i in range(2)]
    torch.manual_seed(2)
    first = [mod.init_state(batch_size=8, device="cuda", dtype=dtype) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def run(x, s):
        out = [mod.prefill_chunked(x[:, :280], s, block_size=40)[0]]
        return out + [mod.step(x[:, t:t + 1].contiguous(), s)[0] for t in range(280, 300)]

    def side_by_side(calls):
        torch.cuda.synchronize()
        for st in streams:
            with torch.cuda.stream(st):
                torch.cuda._sleep(2_000_000)
        out = []
        for st, call in zip(streams, calls):
            with torch.cuda.stream(st):
                out.append(call())
        torch.cuda.synchronize()
        return out

    ends = [_deep_copy_state(s) for s in first]
    want = [run(x, s) for x, s in zip(xs, ends)]
    for _ in range(4):
        states = [_deep_copy_state(s) for s in first]
        got = side_by_side([lambda x=x, s=s: run(x, s) for x, s in zip(xs, states)])
        for a, b, p, q in zip(got, want, states, ends):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
            assert all(torch.equal(getattr(p, f), getattr(q, f)) for f in FIELDS)
    graphs = []
    for x, s in zip(xs, ends):
        xt = x[:, :1].contiguous()
        g = torch.cuda.CUDAGraph()
        arena = s._arena.clone()
        with torch.cuda.graph(g):
            y = mod.step(xt, s)[0]
        g.replay()
        torch.cuda.synchronize()
        graphs.append((g, y, y.clone(), s, arena, s._arena.clone(), xt))
    for _ in range(10):
        for g, y, ref, s, arena, after, xt in graphs:
            s._arena.copy_(arena)
            y.zero_()
        side_by_side([e[0].replay for e in graphs])
        for g, y, ref, s, arena, after, xt in graphs:
            assert torch.equal(y, ref) and torch.equal(s._arena, after)
    assert mod.device_status() == 0


@pytest.mark.gpu
def test_a_capture_without_copies_quantises_each_weight_once(monkeypatch):
    """A first call inside a capture puts into the graph one quantisation of each weight for each time it is used."""
    from coda_gqa_l_b200 import attention
    dtype, kw = SHAPES[1]
    mod = layer(kw, dtype)
    x = hidden(2, 20, kw["embed_dim"], dtype, 3)
    torch.manual_seed(2)
    s = mod.init_state(batch_size=2, device="cuda", dtype=dtype)
    rows = []
    inner = attention.quantize_int8
    monkeypatch.setattr(attention, "quantize_int8", lambda t: rows.append(t.shape) or inner(t))
    heads = mod.num_heads * mod.head_dim
    weights = [(mod.embed_dim, heads)]
    for call in (lambda: mod.prefill_chunked(x, s, block_size=32), lambda: mod.step(x[:, :1].contiguous(), s)):
        rows.clear()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        assert len([r for r in rows if len(r) == 2]) == 2 and sum(r in weights for r in rows) == 1, rows


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kw", SHAPES[:2])
@pytest.mark.parametrize("int8", [True, False])
def test_an_output_bias_is_added_beside_a_residual(dtype, kw, int8):
    """Prefill with the residual taken by the output projection, and the captured step of a stack, with a bias there: what the
    layer gives plus the residual (a rounding more)."""
    from coda_gqa_l_b200 import CoDAStack, _deep_copy_state
    mod = layer(kw, dtype, int8=int8)
    with torch.no_grad():
        mod.o_proj.bias = torch.nn.Parameter(torch.linspace(-8, 8, kw["embed_dim"], device="cuda").to(dtype))
    x = hidden(2, 90, kw["embed_dim"], dtype, 3)
    torch.manual_seed(2)
    s1 = mod.init_state(batch_size=2, device="cuda", dtype=dtype)
    s2 = _deep_copy_state(s1)

    def near(got, y, res):
        # the plain sum rounds twice and another GEMM may have run: three half steps of either term, fp32 sums of 512 terms
        u = torch.finfo(dtype).eps / 2
        bound = (4 * u + 2.0 ** -14) * (y.double().abs() + res.double().abs() + 1)
        assert bool(((got.double() - y.double() - res.double()).abs() <= bound).all()), float((got.double() - y.double() - res.double()).abs().max())

    near(mod.prefill_chunked_residual(x[:, :80], s1, block_size=16), mod.prefill_chunked(x[:, :80], s2, block_size=16)[0], x[:, :80])
    st = CoDAStack([mod])
    for t in range(80, 84):
        xt = x[:, t:t + 1].contiguous()
        near(st.step_graph(xt, [s1]), mod.step(xt, s2)[0], xt)


@pytest.mark.parametrize("int8", [True, False])
def test_a_used_layer_can_be_copied_and_saved(int8, monkeypatch):
    """After the eager step's addresses were gathered: a deep copy and a saved and loaded layer have the parameters and
    switches, and make their own copies of the weights."""
    import copy
    import io
    mod = on_cpu(monkeypatch)
    mod.use_int8_projections = int8
    gather = lambda m: (m._int8_bundle if int8 else m._decode_bundle)(torch.device("cpu"), torch.float32)  # noqa: E731
    with torch.no_grad():
        mine = gather(mod)
        buf = io.BytesIO()
        torch.save(mod, buf)
        buf.seek(0)
        for other in (copy.deepcopy(mod), torch.load(buf, weights_only=False)):
            assert other.use_int8_projections == int8
            for (n, p), (m, q) in zip(mod.named_parameters(), other.named_parameters()):
                assert n == m and torch.equal(p, q) and p.data_ptr() != q.data_ptr()
            theirs = gather(other)
            assert theirs["layer"].bias != mine["layer"].bias
            other.o_proj.weight.mul_(2.0)
            assert gather(other) is not theirs and gather(mod) is mine


@pytest.mark.gpu
def test_a_used_stack_can_be_copied():
    """A stack whose step has been captured: the copy captures its own and gives the same results."""
    import copy

    from coda_gqa_l_b200 import _deep_copy_state
    dtype, kw = SHAPES[1]
    st = stack(kw, dtype, 2, True)
    x = hidden(2, 6, kw["embed_dim"], dtype, 3)
    torch.manual_seed(2)
    s1 = st.init_states(batch_size=2, device="cuda", dtype=dtype)
    st.step_graph(x[:, :1], s1)
    st.step(x[:, 1:2], s1)
    other = copy.deepcopy(st)
    s2 = [_deep_copy_state(s) for s in s1]
    for t in range(2, 6):
        a, b = st.step_graph(x[:, t:t + 1], s1), other.step_graph(x[:, t:t + 1], s2)
        torch.cuda.synchronize()
        assert torch.equal(a, b)
    with torch.no_grad():
        other.layers[0].o_proj.weight.mul_(-1.0)
    a, b = st.step_graph(x[:, :1], s1), other.step_graph(x[:, :1], s2)
    torch.cuda.synchronize()
    assert not torch.equal(a, b)


def test_copies_that_a_capture_used_stay(monkeypatch):
    """Derived copies made before a capture are what the graph reads: another set made later does not free them."""
    import weakref

    from coda_gqa_l_b200 import attention
    mod = on_cpu(monkeypatch)
    mod.use_int8_projections = True
    cpu = torch.device("cpu")

    def made():
        mod._int8_weights()
        t = [mod._fused_weight()[0], mod._skinny_weights()[1], mod._skinny_weights()[2], mod._consts(cpu, torch.float32)[1]]
        return [weakref.ref(x) for x in t], [x.clone() for x in t]

    def change():
        with torch.no_grad():
            set_key(mod)
            mod.o_proj.weight.mul_(0.5)
            mod.theta.add_(0.1)
        return made()

    with torch.no_grad():
        seen, values = made()
        monkeypatch.setattr(attention, "_recording", lambda t: True)
        made()                                             # what a captured call looks up
        monkeypatch.setattr(attention, "_recording", lambda t: False)
        later, _ = change()
        assert all(r() is not None and torch.equal(r(), v) for r, v in zip(seen, values))
        change()
        assert all(r() is not None and torch.equal(r(), v) for r, v in zip(seen, values))
        assert all(r() is None for r in later[1:])         # (made and used outside: not kept)


@pytest.mark.gpu
def test_a_recaptured_stack_keeps_one_set_of_copies():
    """Changed weights make a stack capture again; what the graph before read goes with it."""
    dtype, kw = SHAPES[1]
    st = stack(kw, dtype, 2, True)
    x = hidden(2, 1, kw["embed_dim"], dtype, 3)
    torch.manual_seed(2)
    s = st.init_states(batch_size=2, device="cuda", dtype=dtype)
    sizes = []
    for i in range(6):
        with torch.no_grad():
            for l in st.layers:
                set_key(l)
        st.step_graph(x, s)
        torch.cuda.synchronize()
        sizes.append(torch.cuda.memory_allocated())
        assert all(not l._recorded for l in st.layers)
    assert max(sizes[2:]) - min(sizes[2:]) < 2 ** 20, sizes


@pytest.mark.parametrize("int8", [True, False])
def test_refreshed_weights_are_gathered_again(int8, monkeypatch):
    """Writes past the version counters, announced by refresh_weights: the eager step's copies are those of the new values."""
    mod = on_cpu(monkeypatch)
    mod.use_int8_projections = int8
    gather = lambda: (mod._int8_bundle if int8 else mod._decode_bundle)(torch.device("cpu"), torch.float32)  # noqa: E731
    with torch.no_grad():
        last = gather()
        for p in (mod.q_proj.weight, mod.o_proj.weight):
            p.data.mul_(-2.0)
        mod.refresh_weights()
        now = gather()
        assert now is not last
        if int8:
            assert torch.equal(now["w"][2].scale, mod.o_proj.weight.abs().amax(1) / 127)
        else:
            assert torch.equal(now["w_out_t"], mod.o_proj.weight.t()) and torch.equal(now["w_in_t"], mod._fused_weight()[0].t())
