"""Lists of tensors at the end of a training step (tensor_list.hip, ops.tensor_list / grad_norm / clip_grads / adam, bfsr_amd.optim): refusals and host logic on
the CPU, the kernels against plain 64-bit arithmetic on the GPU.

Tolerances count roundings: u = 2^-24 is one of fp32, half(t) one of the tensor's type, relative to the value; tiny(t) is half of the type's smallest step."""
import copy
import ctypes as C
import math

import pytest
import torch

from bfsr_amd import _lib, ops as O, optim

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
CPU = torch.device("cpu")


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}[t]


# ---- CPU: what is refused, before anything reaches a device --------------------------------------------------------------------------
@pytest.mark.parametrize("bad, error", [
    (torch.zeros(3), TypeError), ([1.0], TypeError), ([torch.zeros(3, dtype=torch.float64)], ValueError), ([torch.zeros(3, dtype=torch.int32)], ValueError),
    ([torch.zeros(4, 4)[:, :2]], ValueError), ([torch.zeros(3, 1).expand(3, 4)], ValueError), ([torch.zeros(8)[::2]], ValueError),
    ([torch.zeros(3).to_sparse()], ValueError), ([torch.zeros(3, device="meta")], ValueError),
    ([torch.zeros(3, dtype=torch.complex64).conj().imag], ValueError)])
def test_list_column_refuses(bad, error):
    with pytest.raises(error):
        O.list_column(bad, CPU, "x")


def test_list_column_takes_any_dense_order():
    w = torch.zeros(4, 3, 5, 2)
    good = [w, w.to(memory_format=torch.channels_last), w.permute(3, 1, 0, 2), torch.zeros(()), torch.zeros(0, 3), torch.zeros(7)[3:], torch.zeros(3, 0).t(),
            torch.zeros(2, 3, dtype=BF16), torch.nn.Parameter(torch.zeros(2))]
    got = O.list_column(good, CPU, "x")
    assert [g.data_ptr() for g in got] == [g.data_ptr() for g in good] and not any(g.requires_grad for g in got)
    O.list_column([w.permute(3, 1, 0, 2)], CPU, "x", like=[torch.empty_like(w).permute(3, 1, 0, 2)])
    for other in (w.to(memory_format=torch.channels_last), torch.zeros(4, 3, 10)):
        with pytest.raises(ValueError):
            O.list_column([other], CPU, "x", like=[w])
    with pytest.raises(ValueError):
        O.list_column([w, w], CPU, "x", like=[w])
    O.list_column([torch.zeros(4, 1, 3, 3).to(memory_format=torch.channels_last)], CPU, "x", like=[torch.zeros(4, 1, 3, 3).contiguous().to(memory_format=torch.channels_last)])


def test_spans_find_overlaps():
    a = torch.zeros(100)
    pieces = lambda ts: (O._addresses(ts), O._bytes(ts))                    # noqa: E731
    spans = lambda ts: O.Spans(*pieces(ts), "x")                            # noqa: E731
    spans([a[:10], a[10:20], a[50:], a[30:30], a[20:50]])
    for pair in ([a, a], [a[:10], a[9:20]], [a, a[40:41]], [a[5:6], a[:10]]):
        with pytest.raises(ValueError):
            spans(pair)
    s = spans([a[10:20], a[40:60]])
    assert not s.meet(*pieces([])) and not s.meet(*pieces([a[:10], a[20:40], a[60:], a[15:15]]))
    for t in (a[9:11], a[19:25], a[30:41], a[59:], a[12:13], a):
        assert s.meet(*pieces([a[:5], t]))
    assert not spans([]).meet(*pieces([a]))


def test_numbers_out_of_range_are_refused():
    assert O._norm_type("inf") == O._norm_type(math.inf) == 1 and O._norm_type(2) == O._norm_type(2.0) == 0
    for v in (1.0, 0, -1, math.nan, 3.5, None):
        with pytest.raises(ValueError):
            O._norm_type(v)
    for v in (-1e-30, math.nan, -math.inf):
        with pytest.raises(ValueError):
            O._at_least_0(v, "x")
    with pytest.raises(ValueError):
        O._at_least_0(1.0, "beta", 1.0)
    with pytest.raises(TypeError):
        O._at_least_0(torch.ones(()), "x")
    assert O._at_least_0(0.999, "beta", 1.0) == 0.999 and O._at_least_0(math.inf, "x") == math.inf
    for t in (torch.zeros(2), torch.zeros((), dtype=torch.float64), 1.0, torch.zeros((), device="meta")):
        with pytest.raises(ValueError):
            O._one_float(t, CPU, "x")


def test_c_entries_refuse_before_a_launch():
    lib = _lib.load()
    chunk = lib.bfsr_list_chunk(1000)
    assert chunk > 0 and chunk % 1024 == 0 and lib.bfsr_list_chunk(-1) == -1 and lib.bfsr_list_work(-1) == -1 and lib.bfsr_list_work(5) > lib.bfsr_list_work(0) > 0
    one = (C.c_void_p * 1)(4096)
    cols = lambda n: (C.c_void_p * n)(*[C.addressof(one)] * n)             # noqa: E731
    size, kind = (C.c_longlong * 1)(8), (C.c_int * 1)(0)

    def write(ncols=1, c=None, sizes=size, types=kind, n=1, ch=chunk, rows=4096, chunks=4096):
        return lib.bfsr_list_write(cols(5) if c is None else c, ncols, sizes, types, n, ch, rows, chunks, None)

    null = (C.c_void_p * 1)(0)
    assert write(ncols=3) == write(ncols=0) == write(n=0) == write(ch=0) == write(ch=1000) == write(rows=None) == write(chunks=None) == -1
    assert write(sizes=(C.c_longlong * 1)(-1)) == write(types=(C.c_int * 1)(3)) == write(types=(C.c_int * 1)(3 << 4)) == write(types=(C.c_int * 1)(-1)) == -1
    assert write(c=(C.c_void_p * 1)(0)) == write(c=(C.c_void_p * 1)(C.addressof(null))) == -1
    assert write(ncols=5, sizes=(C.c_longlong * 1)(0), c=(C.c_void_p * 5)(*[C.addressof(one)] * 4 + [C.addressof(null)])) == -1
    assert write(sizes=(C.c_longlong * 1)(chunk << 24)) == write(sizes=(C.c_longlong * 1)((1 << 63) - 1)) == -1
    assert lib.bfsr_pointer_write(None, 1, 4096, None) == lib.bfsr_pointer_write(one, 0, 4096, None) == lib.bfsr_pointer_write(one, 1, None, None) == -1
    a, h = _lib.BfsrListArgs(), _lib.BfsrAdamArgs()
    good = dict(rows=4096, chunks=4096, n=1, count=1, chunk=chunk, work=4096, norm=4096)
    for bad in (dict(rows=None), dict(chunks=None), dict(n=0), dict(count=-1), dict(count=1 << 24), dict(chunk=0), dict(chunk=1000), dict(work=None, count=1000), dict(norm=None)):
        for k, v in dict(good, **bad).items():
            setattr(a, k, v)
        h.beta1, h.beta2, h.max_norm = 0.9, 0.999, 1.0
        assert lib.bfsr_norm_work(1000) > 0 == lib.bfsr_norm_work(1) and lib.bfsr_norm_work(-1) == -1
        assert lib.bfsr_grad_norm(C.byref(a), None) == lib.bfsr_clip_grads(C.byref(a), 1.0, None) == lib.bfsr_adam_step(C.byref(a), C.byref(h), None) == -1, bad
    for k, v in good.items():
        setattr(a, k, v)
    assert lib.bfsr_grad_norm(None, None) == lib.bfsr_clip_grads(C.byref(a), -1.0, None) == lib.bfsr_clip_grads(C.byref(a), math.nan, None) == -1
    for name, v in (("beta1", 1.0), ("beta2", -0.1), ("eps", -1.0), ("weight_decay", math.nan), ("beta1", math.nan)):
        h = _lib.BfsrAdamArgs(beta1=0.9, beta2=0.999, max_norm=-1.0)
        setattr(h, name, v)
        assert lib.bfsr_adam_step(C.byref(a), C.byref(h), None) == -1, name


def test_optimizer_host_side():
    """Argument checks, state dicts of torch's Adam in and out, copies -- no step."""
    p = [torch.nn.Parameter(torch.randn(4, 3)), torch.nn.Parameter(torch.randn(5).bfloat16())]
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(weight_decay=-0.1), dict(max_grad_norm=-1.0), dict(max_grad_norm=math.nan)):
        with pytest.raises(ValueError):
            optim.Adam(p, **bad)
    q = [torch.nn.Parameter(t.detach().clone()) for t in p]
    ref = torch.optim.Adam(q, lr=0.1)
    for _ in range(2):
        for t in q:
            t.grad = torch.ones_like(t)
        ref.step()
    sd = ref.state_dict()
    sd["state"][1]["exp_avg"] = torch.full((5,), 1.0 + 2.0 ** -20)          # fp32 moments of a bf16 parameter stay fp32
    own = optim.Adam(p, lr=0.5, max_grad_norm=2.0)
    own.load_state_dict(sd)
    assert own.param_groups[0]["lr"] == 0.1 and not own.param_groups[0]["decoupled_weight_decay"]
    assert float(own.state[p[0]]["step"]) == 2.0 and own.state[p[1]]["exp_avg"].dtype == F32 and float(own.state[p[1]]["exp_avg"][0]) == 1.0 + 2.0 ** -20
    assert torch.equal(own.state[p[0]]["exp_avg"], sd["state"][0]["exp_avg"]) and own.state[p[0]]["exp_avg"].data_ptr() != sd["state"][0]["exp_avg"].data_ptr()
    back = torch.optim.Adam(q, lr=1.0)
    back.load_state_dict(own.state_dict())
    assert torch.equal(back.state[q[0]]["exp_avg_sq"], sd["state"][0]["exp_avg_sq"])
    twin = copy.deepcopy(own)
    assert twin.max_grad_norm == 2.0 and twin._plans == {} and twin._ops is None
    with pytest.raises(ValueError):
        own.load_state_dict(torch.optim.Adam(q, lr=7.0, amsgrad=True).state_dict())
    assert own.param_groups[0]["lr"] == 0.1 and float(own.state[p[0]]["step"]) == 2.0
    p[0].grad = torch.ones_like(p[0])
    with pytest.raises(ValueError):
        optim.Adam(p).step()                                                # no CPU path
    with pytest.raises(ValueError):
        optim.clip_grad_norm(p, 1.0)
    assert float(optim.clip_grad_norm([torch.zeros(2)], 1.0)) == 0.0        # nothing has a gradient
    p[0].grad = torch.ones_like(p[0]).to_sparse()
    with pytest.raises(RuntimeError):
        optim.Adam(p).step()


def test_train_step_clips_with_the_models_ops(golden_dir):
    """train_step(max_grad_norm=): the gradients go through the frozen model's ops, and the norm comes back."""
    from cpu_ops import CpuOps
    from test_linf_cpu import run_train_step_case
    import bfsr_amd.linf.train as train

    class Double(CpuOps):
        def clip_grads(self, tensors, max_norm, norm_type=2.0):
            tensors = O.list_column(tensors, CPU, "x")
            norm = torch.sqrt(sum(t.double().square().sum() for t in tensors)).float()
            for t in tensors:
                t.mul_((max_norm / (norm + 1e-6)).clamp(max=1.0))
            return norm

    plain, prior, _ = run_train_step_case(golden_dir, Double())
    assert "grad_norm" not in plain
    want = torch.sqrt(sum(p.grad.double().square().sum() for p in prior.parameters()))
    step, had = train.train_step, [p.grad.clone() for p in prior.parameters()]
    try:
        train.train_step = lambda *a, **k: step(*a, max_grad_norm=float(want) / 3, **k)
        out, clipped, _ = run_train_step_case(golden_dir, Double())
    finally:
        train.train_step = step
    assert abs(out["grad_norm"] - float(want)) <= 1e-6 * float(want)
    share = float(want) / 3 / (float(want) + 1e-6)
    for a, b in zip(had, clipped.parameters()):
        assert (a * share - b.grad).abs().max() <= 1e-5 * a.abs().max()


# ---- GPU --------------------------------------------------------------------------------------------------------------------------------
gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _grad():
    """Other test modules turn gradients off for the whole process."""
    with torch.enable_grad():
        yield


@pytest.fixture(scope="module")
def hip():
    return O.HipOps("cuda:0")


SIZES = [(1,), (2,), (3,), (0,), (4,), (5, 1), (63,), (64,), (), (1023,), (1024,), (1025,), (4095,), (64, 64), (4097,), (16, 9, 3, 3), (37, 37, 3, 3), (12289,)]


SHORT = [(1,), (0,), (5, 1), (63,), (), (1025,), (2048,), (2051,)]          # one workgroup clips it, and takes a step, by itself
LONG = SIZES + [(300001,)]                                                  # ... and several


def make(seed, shapes=SIZES, types=(F32,), scale=1.0, lead=0):
    """Tensors on the GPU, the types in turn; `lead` > 0: views that start `lead` elements into a buffer (no alignment but the element's)."""
    g = torch.Generator().manual_seed(seed)
    got = []
    for k, s in enumerate(shapes):
        t = (torch.randn(s, generator=g) * scale).to(types[k % len(types)])
        base = torch.full((t.numel() + lead + 1,), 77.0, dtype=t.dtype, device="cuda:0")
        v = base[lead:lead + t.numel()].view(s)
        v.copy_(t)
        got.append(v)
    return got


def doubles(ts):
    return [t.detach().cpu().double() for t in ts]


def norm64(ts, kind=2.0):
    flat = torch.cat([t.reshape(-1) for t in ts] or [torch.zeros(0, dtype=torch.float64)])
    return float(flat.abs().max() if kind == math.inf else flat.square().sum().sqrt()) if flat.numel() else 0.0


def near_norm(got, want, n=1 << 20):
    """One rounding to fp32, and the order of a 64-bit sum of n terms."""
    assert got.shape == () and got.dtype == F32
    assert abs(float(got) - want) <= want * (U + n * 2.0 ** -53) + tiny(F32), (float(got), want)


def near_clipped(got, grads, share):
    for k, (a, g) in enumerate(zip(got, grads)):
        want = g * share
        bound = want.abs() * (half(a.dtype) + 3 * U) + tiny(a.dtype)        # the share's rounding, the product's, and the type's
        assert bool(((a.cpu().double() - want).abs() <= bound).all()), (k, tuple(a.shape), a.dtype)


TYPES = [(F32,), (F16,), (BF16,), (F32, BF16, F16)]


@gpu
@pytest.mark.parametrize("lead", [0, 1, 3])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_grad_norm(hip, types, kind, lead):
    ts = make(1, types=types, lead=lead)
    near_norm(hip.grad_norm(hip.tensor_list(ts), kind), norm64(doubles(ts), kind))
    out = torch.zeros(1, device="cuda:0")
    assert hip.grad_norm(hip.tensor_list(ts), kind, out=out) is out
    near_norm(out[0], norm64(doubles(ts), kind))


@gpu
@pytest.mark.parametrize("shapes", [[(1,)], [(0,)], [(0,), (1,)], [()], [(100000,)], [(3, 7)] * 1500, [(262144,)] * 5 + [(1,)] * 300, [(4, 3, 3, 3)] * 61, [(4,)] * 62])
def test_norm_and_clip_of_many_and_few(hip, shapes):
    ts = make(2, shapes=shapes, types=(F32, F32, BF16))
    want = doubles(ts)
    for kind in (2.0, math.inf):
        norm = norm64(want, kind)
        near_norm(hip.grad_norm(hip.tensor_list(ts), kind), norm, 1 << 22)
        into = [torch.full_like(t, 9.0) for t in ts]
        most = norm / 3 + 1e-3
        near_norm(hip.clip_grads(hip.tensor_list(ts, out=into), most, kind), norm, 1 << 22)
        near_clipped(into, want, min(1.0, most / (norm + 1e-6)))
        assert all(torch.equal(a, b.to(a.dtype)) for a, b in zip(doubles(ts), want))


@gpu
@pytest.mark.parametrize("lead", [0, 1])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("shapes", [SHORT, LONG])
def test_clip_in_place(hip, shapes, types, kind, lead):
    ts = make(3, shapes, types=types, lead=lead, scale=0.5)
    want, versions = doubles(ts), [t._version for t in ts]
    norm = norm64(want, kind)
    near_norm(hip.clip_grads(hip.tensor_list(ts), 0.25 * norm, kind), norm)
    near_clipped(ts, want, 0.25 * norm / (norm + 1e-6))
    assert all(t._version == v + 1 for t, v in zip(ts, versions))
    for t in ts:                                                            # nothing outside the views
        base = t._base if t._base is not None else t
        assert float(base.reshape(-1)[-1]) == 77.0 and (not lead or float(base.reshape(-1)[0]) == 77.0)
    had = doubles(ts)
    near_norm(hip.clip_grads(hip.tensor_list(ts), 1e9, kind), norm64(had, kind))        # within the bound: not a bit changes
    assert all(torch.equal(a, b) for a, b in zip(had, doubles(ts)))


@gpu
def test_orders_of_axes(hip):
    w = make(4, shapes=[(8, 6, 5, 5)] * 3)
    ts = [w[0].to(memory_format=torch.channels_last), w[1].permute(2, 0, 3, 1), w[2].transpose(0, 1)]
    want = doubles(ts)
    norm = norm64(want)
    near_norm(hip.clip_grads(hip.tensor_list(ts), 1.0), norm)
    near_clipped(ts, want, 1.0 / (norm + 1e-6))


@gpu
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_far_and_near_magnitudes(hip, kind):
    """Squares that overflow or vanish in 32 bits."""
    for scale in (1e30, 1e-30, 1e-40):
        ts = make(5, scale=scale)
        want = doubles(ts)
        norm = norm64(want, kind)
        near_norm(hip.grad_norm(hip.tensor_list(ts), kind), norm)
        near_norm(hip.clip_grads(hip.tensor_list(ts), 1.0, kind), norm)
        near_clipped(ts, want, min(1.0, 1.0 / (norm + 1e-6)))


@gpu
@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("at", [0, 7, 16])
@pytest.mark.parametrize("shapes", [SIZES, LONG])
def test_not_finite(hip, shapes, kind, bad, at):
    ts = make(6, shapes, types=(F32, BF16, F16))
    ts[at].reshape(-1)[-1] = bad
    norm = hip.grad_norm(hip.tensor_list(ts), kind)
    assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
    hip.clip_grads(hip.tensor_list(ts), 1.0, kind)
    for k, t in enumerate(ts):
        flat = t.reshape(-1)
        if math.isnan(bad):
            assert bool(flat.isnan().all())
        else:
            assert bool(flat[-1:].isnan().all()) == (k == at or not t.numel()) and not bool(flat[:-1].any())


@gpu
def test_nan_survives_larger_numbers(hip):
    """The largest magnitude is NaN where one is, before or behind infinities, in whichever lane."""
    for size in (1, 5, 70, 5000, 1 << 17):
        for at in (0, size // 2, size - 1):
            t = torch.full((size,), math.inf, device="cuda:0")
            t[at] = math.nan
            assert math.isnan(float(hip.grad_norm(hip.tensor_list([t]), math.inf)))


@gpu
def test_offsets_beyond_32_bits(hip):
    n = (1 << 32) + 4099
    t = torch.zeros(n, dtype=BF16, device="cuda:0")
    t[5], t[1 << 31], t[(1 << 32) + 1], t[n - 1] = 1.0, 2.0, 4.0, 10.0
    one = torch.ones(3, device="cuda:0")
    tl = hip.tensor_list([t, one])
    near_norm(hip.clip_grads(tl, 1.0), math.sqrt(1 + 4 + 16 + 100 + 3), 1)
    got = [float(t[k]) for k in (5, 1 << 31, (1 << 32) + 1, n - 1)]
    share = 1.0 / (math.sqrt(124) + 1e-6)
    assert all(abs(a - b * share) <= b * share * (2.0 ** -8 + 3 * U) for a, b in zip(got, (1, 2, 4, 10)))
    assert float(hip.grad_norm(tl, math.inf)) == max(got + [float(one[0])])


@gpu
@pytest.mark.parametrize("types", TYPES)
def test_plain_lists(hip, types):
    """A list of tensors in place of a handle, on any stream."""
    ts = make(9, types=types)
    want = doubles(ts)
    near_norm(hip.grad_norm(ts), norm64(want))
    near_norm(hip.grad_norm(iter(ts), math.inf), norm64(want, math.inf))
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        norm = hip.clip_grads(ts, 1.0)
    torch.cuda.synchronize()
    near_norm(norm, norm64(want))
    near_clipped(ts, want, min(1.0, 1.0 / (norm64(want) + 1e-6)))
    assert float(hip.grad_norm([])) == 0.0
    empty = [torch.zeros(0, device="cuda:0")] * 2
    assert float(hip.grad_norm(empty)) == 0.0 == float(hip.clip_grads(hip.tensor_list(empty), 1.0, math.inf))


@gpu
@pytest.mark.parametrize("most", [0.0, math.inf])
def test_extreme_bounds(hip, most):
    ts = make(10, types=(F32, BF16))
    want = doubles(ts)
    hip.clip_grads(ts, most)
    near_clipped(ts, want, 0.0 if most == 0.0 else 1.0)
    zeros = [torch.zeros(5, device="cuda:0")]
    assert float(hip.clip_grads(zeros, most)) == 0.0 and not bool(zeros[0].any())


@gpu
def test_same_bits_every_time(hip):
    ts = make(7, shapes=[(100003,), (512, 300), (7,)] * 20, types=(F32, BF16))
    tl = hip.tensor_list(ts)
    got = {float(hip.grad_norm(tl)) for _ in range(20)} | {float(hip.grad_norm(hip.tensor_list(ts)))}
    assert len(got) == 1


@gpu
def test_lists_are_refused(hip):
    a, b = make(8, shapes=[(8,), (8,)])
    for bad in ([a, a], [a, b, a[2:4]], [a.cpu()], [a.double()], [a[::2]]):
        with pytest.raises(ValueError):
            hip.tensor_list(bad)
    for out in ([b], [b, b], [a, b], [torch.empty_like(a), torch.empty(9, device="cuda:0")], [torch.empty_like(a), torch.empty_like(b, dtype=F16)]):
        with pytest.raises(ValueError):
            hip.tensor_list([a, b], out=out)
    tl = hip.tensor_list([a])
    for bad, error in ((a, TypeError), ([a, 1.0], TypeError), ([a, a], ValueError)):
        for call in (hip.grad_norm, lambda t: hip.clip_grads(t, 1.0), hip.tensor_list):
            with pytest.raises(error):
                call(bad)
    with pytest.raises(ValueError):
        O.HipOps("cuda:0").grad_norm(tl)
    for call in (lambda: hip.grad_norm(tl, 1.0), lambda: hip.clip_grads(tl, -1.0), lambda: hip.clip_grads(tl, math.nan), lambda: hip.grad_norm(tl, out=torch.zeros(2, device="cuda:0")),
                 lambda: hip.grad_norm(tl, out=torch.zeros(1))):
        with pytest.raises(ValueError):
            call()
    empty = hip.tensor_list([])
    assert float(hip.grad_norm(empty)) == 0.0 == float(hip.clip_grads(empty, 1.0)) and float(hip.grad_norm(empty, out=torch.ones((), device="cuda:0"))) == 0.0


# ---- Adam
def adam64(p, g, m, v, t, lr, betas, eps, wd, decoupled, share):
    """One step in 64 bits, and how far 32 bits may be from it: every rounding of the kernel's formula, carried to the end."""
    b1, b2 = betas
    x, ex = g * share, (g * share).abs() * 2 * U
    ep = 0.0
    if wd and decoupled:
        p = p * (1 - lr * wd)
        ep = p.abs() * 2 * U
    elif wd:
        ex = ex + (wd * p).abs() * U
        x = x + wd * p
        ex = ex + x.abs() * U
    low = 2.0 ** -148                                                       # steps among the smallest numbers are absolute
    m1 = b1 * m + (1 - b1) * x
    em = (b1 * m).abs() * U + ((1 - b1) * x).abs() * 2 * U + (1 - b1) * ex + m1.abs() * U + low
    v1 = b2 * v + (1 - b2) * x * x
    ev = (b2 * v).abs() * U + (1 - b2) * x * x * 3 * U + 2 * (1 - b2) * x.abs() * ex + (1 - b2) * ex * ex + v1 * U + low
    size, root = lr / (1 - b1 ** t), 1 / math.sqrt(1 - b2 ** t)
    r = v1.sqrt()
    er = torch.minimum(ev / (2 * r).clamp_min(1e-300), ev.sqrt()) * 1.01 + r * 2 * U     # |sqrt(a) - sqrt(b)| is at most both
    d = r * root + eps
    ed = er * root * 1.01 + r * root * U + eps * U + d * U
    q = m1 / d
    eq = em / (d - ed).clamp_min(1e-300) + q.abs() * ed / (d - ed).clamp_min(1e-300) + q.abs() * 2 * U
    p1 = p - size * q
    ep = ep + size * eq * 1.01 + (size * q).abs() * 2 * U + p1.abs() * U + low
    return (p1, m1, v1), (ep, em, ev)


def adam_case(seed, shapes, types, grad_types, lead=0, steps=(0.0, 1.0, 10.0, 999.0)):
    p = make(seed, shapes, types, 0.1, lead)
    g = make(seed + 1, shapes, grad_types, 0.02, lead)
    m = make(seed + 2, shapes, (F32,), 0.01, lead)
    v = [t.square_() for t in make(seed + 3, shapes, (F32,), 0.02, lead)]
    step = torch.tensor([steps[k % len(steps)] for k in range(len(shapes))], device="cuda:0")
    for k in range(len(shapes)):
        if float(step[k]) == 0:
            m[k].zero_()
            v[k].zero_()
    return p, g, m, v, step


def check_adam(hip, p, g, m, v, step, plan=None, share=1.0, norm=None, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, wd=0.0, decoupled=False, **kw):
    had = [doubles(c) for c in (p, g, m, v)]
    t = (step + 1).tolist()
    plan = plan or hip.adam(p, g, m, v, step)
    got = plan.run(lr, betas, eps, wd, decoupled, **kw)
    assert (got is None) == (norm is None)
    if norm is not None:
        near_norm(got, norm)
    assert step.tolist() == t
    rate = float(lr)
    for k in range(len(p)):
        want, bound = adam64(had[0][k], had[1][k], had[2][k], had[3][k], t[k], rate, betas, eps, wd, decoupled, share)
        for name, a, w, b in zip("pmv", (p[k], m[k], v[k]), want, bound):
            b = b + w.abs() * (half(a.dtype) * 1.01 if a.dtype != F32 else 0.0) + tiny(a.dtype)
            off = (a.cpu().double() - w).abs()
            assert bool((off <= b).all()), (k, tuple(a.shape), name, a.dtype, float((off / b).max()))
        assert torch.equal(g[k].cpu().double(), had[1][k])
    return plan


@gpu
@pytest.mark.parametrize("lead", [0, 1])
@pytest.mark.parametrize("types, grad_types", [((F32,), (F32,)), ((BF16,), (BF16,)), ((F16,), (F16,)), ((F32,), (BF16,)), ((F32,), (F16,)), ((F32, BF16, F16), (F16, F32, BF16, BF16))])
@pytest.mark.parametrize("shapes", [SHORT, SIZES])
def test_adam_types(hip, shapes, types, grad_types, lead):
    case = adam_case(20, shapes, types, grad_types, lead)
    plan = check_adam(hip, *case)
    check_adam(hip, *case, plan=plan, wd=0.1)
    for c in (case[0], case[2]):
        for t in c:
            assert float(t._base.reshape(-1)[-1]) == 77.0


@gpu
@pytest.mark.parametrize("wd, decoupled", [(0.0, False), (0.3, False), (0.3, True)])
@pytest.mark.parametrize("most", [None, 0.3, 1e6])
@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("shapes", [SHORT, SIZES])
def test_adam_decay_and_clipping(hip, shapes, wd, decoupled, most, kind):
    case = adam_case(30, shapes, (F32, BF16), (F32, BF16, F32))
    norm = norm64(doubles(case[1]), kind)
    scaled = most if most != 0.3 else 0.3 * norm
    share = 1.0 if most is None else min(1.0, scaled / (norm + 1e-6))
    check_adam(hip, *case, share=share, norm=None if most is None else norm, wd=wd, decoupled=decoupled, max_norm=scaled, norm_type=kind)


@gpu
@pytest.mark.parametrize("betas, eps, lr", [((0.0, 0.0), 1e-8, 1e-2), ((0.5, 0.9999), 1e-3, 1.0), ((0.99, 0.5), 1e-15, 1e-5), ((0.9, 0.999), 1.0, 0.0)])
def test_adam_numbers(hip, betas, eps, lr):
    check_adam(hip, *adam_case(40, SIZES, (F32,), (F32,)), betas=betas, eps=eps, lr=lr)


LARGE = [(3500017,), (33,), (2999, 1001), (0,), (3000000,), (1,)]           # more than the shared cache is counted on for: read and written past it


@gpu
@pytest.mark.parametrize("lead", [0, 1])
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_large_lists(hip, kind, lead):
    ts = make(45, LARGE * 3, (F32, BF16, F16, F32), 0.1, lead)
    want = doubles(ts)
    norm = norm64(want, kind)
    into = [torch.full_like(t, 7.0) for t in ts]
    tl = hip.tensor_list(ts, out=into)
    assert tl.bytes > 128 << 20
    near_norm(hip.grad_norm(tl, kind), norm, 1 << 25)
    near_norm(hip.clip_grads(tl, norm / 3, kind), norm, 1 << 25)
    near_clipped(into, want, norm / 3 / (norm + 1e-6))
    del ts, into, tl, want
    case = adam_case(46, LARGE, (F32, F32, BF16, F32), (F32, BF16, F16, F32), lead)
    norm = norm64(doubles(case[1]), kind)
    plan = check_adam(hip, *case, share=0.5 * norm / (norm + 1e-6), norm=norm, max_norm=0.5 * norm, norm_type=kind, wd=0.1, decoupled=bool(lead))
    assert plan.bytes > 128 << 20
    base = case[0][0]._base
    assert float(base.reshape(-1)[-1]) == 77.0 and (not lead or float(base.reshape(-1)[0]) == 77.0)


@gpu
def test_adam_many_small_tensors_and_a_list_of_counts(hip):
    p, g, m, v, step = adam_case(50, [(3, 5)] * 700 + [(70000,)], (F32,), (F32,))
    counts = [s.clone() for s in step.unbind()]
    plan = hip.adam(p, g, m, v, counts)
    had = [doubles(c) for c in (p, g, m, v)]
    plan.run(1e-2)
    for k in (0, 1, 61, 62, 63, 480, 699, 700):
        want, bound = adam64(*[h[k] for h in had], float(step[k]) + 1, 1e-2, (0.9, 0.999), 1e-8, 0.0, False, 1.0)
        assert float(counts[k]) == float(step[k]) + 1
        assert bool(((p[k].cpu().double() - want[0]).abs() <= bound[0]).all()), k


@gpu
@pytest.mark.parametrize("shapes", [[(3, 5)] * 500 + [(70000,)], [(3, 5)] * 5 + [(700,)], [(0,)] * 3])
def test_adam_with_other_gradients_rate_and_norm_on_the_device(hip, shapes):
    p, g, m, v, step = adam_case(60, shapes, (F32,), (F32,))
    plan = hip.adam(p, None, m, v, step)
    with pytest.raises(ValueError):
        plan.run(1e-2)
    other = make(66, shapes, (F32,), 0.3, lead=1)
    lr = torch.tensor([0.02], device="cuda:0")
    norm = torch.tensor(8.0, device="cuda:0")
    case = (p, other, m, v, step)
    check_adam(hip, *case, plan=plan, lr=lr, grads=other, max_norm=2.0, grad_norm=norm, norm=8.0, share=2.0 / (8.0 + 1e-6))
    check_adam(hip, *case, plan=plan, lr=lr, grads=other)
    for bad in (other[:-1], [t.half() for t in other], [t.cpu() for t in other], p, [t[:1] for t in other]):
        if bad is not other and not any(t.numel() for t in other) and bad[0].device == other[0].device and len(bad) == len(other) and bad[0].dtype == F32:
            continue                                                        # nothing to tell empty ones apart by
        with pytest.raises(ValueError):
            plan.run(1e-2, grads=bad)
    with pytest.raises(ValueError):
        plan.run(1e-2, grads=other, grad_norm=norm)


@gpu
@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("most", [None, 1.0])
@pytest.mark.parametrize("shapes, at", [(SHORT, 5), (SIZES, 9), ([(3,)] * 400, 9), ([(0,)] * 300 + [(7,)], 300)])
def test_adam_skips_or_takes_what_is_not_finite(hip, shapes, at, bad, most):
    case = adam_case(70, shapes, (F32, BF16), (F32,))
    p, g, m, v, step = case
    g[at].reshape(-1)[2] = bad
    had = [[t.clone() for t in c] for c in (p, m, v)] + [step.clone()]
    plan = hip.adam(*case)
    norm = plan.run(1e-2, max_norm=most, skip_nonfinite=True, weight_decay=0.1)
    assert not math.isfinite(float(norm))
    assert torch.equal(step, had[3]) and all(torch.equal(a, b) for c, h in zip((p, m, v), had) for a, b in zip(c, h))
    plan.run(1e-2, max_norm=most)
    assert bool(p[at].isnan().any()) and torch.equal(step, had[3] + 1)
    g[at].reshape(-1)[2] = 0.5
    for c, h in zip((p, m, v), had):
        for a, b in zip(c, h):
            a.copy_(b)
    check_adam(hip, *case, plan=plan, norm=norm64(doubles(g)), max_norm=most, skip_nonfinite=True,
               share=1.0 if most is None else min(1.0, most / (norm64(doubles(g)) + 1e-6)))


@gpu
def test_adam_is_refused(hip):
    p, g, m, v, step = adam_case(80, [(4,), (5, 3)], (F32,), (F32,))
    wrong = torch.zeros(4, device="cuda:0")
    for args in (([], [], [], [], []), (p, g[:1], m, v, step), (p, g, m, [t.half() for t in v], step), (p, g, m, m, step), (p, p, m, v, step), (p, g, m, v, step[:1]),
                 (p, g, m, v, step.double()), (p, g, m, v, step.view(1, 2)), (p, g, m, v, [step[0], step[0]]), (p, g, [m[0], m[1].t().contiguous().t()], v, step),
                 (p, g, m, v, [wrong, step[0]]), (p, g, m, [v[0], p[1]], step), ([p[0], p[0]], g, m, v, step)):
        with pytest.raises(ValueError):
            hip.adam(*args)
    plan = hip.adam(p, g, m, v, step)
    for kw in (dict(lr=-1.0), dict(lr=torch.zeros(1)), dict(lr=0.1, betas=(1.0, 0.5)), dict(lr=0.1, eps=-1.0), dict(lr=0.1, weight_decay=-1.0), dict(lr=0.1, max_norm=-1.0),
               dict(lr=0.1, norm_type=1.0), dict(lr=0.1, max_norm=1.0, grad_norm=step)):
        with pytest.raises(ValueError):
            plan.run(**kw)


# ---- streams and graphs
@gpu
def test_other_streams_and_two_at_once(hip):
    ts = make(90, shapes=[(1 << 20,), (999,), (512, 777)])
    want = norm64(doubles(ts))
    tl = hip.tensor_list(ts)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [hip.grad_norm(tl) for _ in range(10)]
    torch.cuda.synchronize()
    for a in got:
        near_norm(a, want, 1 << 21)
    with torch.cuda.stream(streams[0]):
        last = hip.grad_norm(tl)
        del tl
        junk = [torch.full((64,), 3, dtype=torch.int64, device="cuda:0") for _ in range(64)]      # memory of the table, if it were free already
    torch.cuda.synchronize()
    near_norm(last, want, 1 << 21)
    del junk


@gpu
def test_captured_norm_and_clip(hip):
    ts = make(91, shapes=[(70001,), (33, 65), (5,)], types=(F32, BF16))
    first = [t.clone() for t in ts]
    tl, two = hip.tensor_list(ts), hip.tensor_list(first)
    with torch.cuda.graph(a := torch.cuda.CUDAGraph()):
        norm = hip.clip_grads(tl, 1.0)
        with pytest.raises(RuntimeError):
            hip.tensor_list(ts)
    with torch.cuda.graph(b := torch.cuda.CUDAGraph()):
        other = hip.grad_norm(two)
    del tl
    for k in range(4):
        for t, f in zip(ts, first):
            t.copy_(f * (k + 1))
        now = doubles(ts)
        a.replay()
        b.replay()
        torch.cuda.synchronize()
        near_norm(norm, norm64(now))
        near_norm(other, norm64(doubles(first)))
        near_clipped(ts, now, min(1.0, 1.0 / (norm64(now) + 1e-6)))
        eager = hip.grad_norm(two)
        assert float(eager) == float(other)


@gpu
def test_captured_adam_follows_the_rate(hip):
    case = adam_case(92, [(3000,), (17, 65), (5,)], (F32, BF16), (F32, F32, BF16), steps=(4.0,))
    p, g, m, v, step = case
    lr = torch.tensor(0.1, device="cuda:0")
    plan = hip.adam(*case)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = plan.run(lr, max_norm=0.5, weight_decay=0.1, decoupled=True)

    class Replay:
        def run(self, *a, **k):
            graph.replay()
            torch.cuda.synchronize()
            return norm

    for k in range(4):
        lr.fill_(0.1 / (k + 1))
        g[0].mul_(1.5)
        n = norm64(doubles(g))
        check_adam(hip, *case, plan=Replay(), lr=float(lr), wd=0.1, decoupled=True, norm=n, share=min(1.0, 0.5 / (n + 1e-6)))
        n = norm64(doubles(g))
        check_adam(hip, *case, plan=plan, lr=float(lr), norm=n, share=min(1.0, 0.5 / (n + 1e-6)), max_norm=0.5)


# ---- the run of them together, as a program has it
class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        torch.manual_seed(5)
        self.a = torch.nn.Conv2d(3, 17, 3, padding=1)
        self.b = torch.nn.Conv2d(17, 17, 3, padding=1, groups=1).to(memory_format=torch.channels_last)
        self.c = torch.nn.Conv2d(17, 3, 1)
        self.unused = torch.nn.Parameter(torch.ones(3))

    def forward(self, x):
        return self.c(torch.relu(self.b(torch.relu(self.a(x)))))


def close_steps(own, ref, lr, steps):
    """Each step's update is at most about lr in size (bounded by 10 lr for any betas used here) and is off by a few dozen roundings of itself and two of the
    parameter; gradients come from the two nets' own parameters, whose difference the tests keep at the level of the roundings by sharing them."""
    for a, b in zip(own, ref):
        b = b.detach().cpu().double()
        assert bool(((a.detach().cpu().double() - b).abs() <= steps * (U * 4 * b.abs() + 64 * U * 10 * lr)).all())


@gpu
@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("decoupled", [False, True])
def test_optimizer_against_torch_in_64_bits(hip, decoupled, groups):
    """optim.Adam on the GPU and torch's Adam / AdamW in float64 on the CPU, given the same gradients; parameters without a gradient keep their count."""
    net, ref = Net().cuda(), Net().double()
    split = lambda n: [dict(params=list(n.parameters())[:3]), dict(params=list(n.parameters())[3:], lr=0.003)] if groups == 2 else list(n.parameters())     # noqa: E731
    own = optim.Adam(split(net), lr=0.01, weight_decay=0.1, decoupled_weight_decay=decoupled, max_grad_norm=0.5, ops=hip)
    theirs = (torch.optim.AdamW if decoupled else torch.optim.Adam)(split(ref), lr=0.01, weight_decay=0.1)
    rates = [torch.optim.lr_scheduler.MultiStepLR(o, [2, 4], 0.5) for o in (own, theirs)]
    for k in range(5):
        own.zero_grad()
        theirs.zero_grad()
        net(torch.randn(2, 3, 16, 16, generator=torch.Generator().manual_seed(k)).cuda()).square().mean().backward()
        if k == 2:
            net.c.bias.grad = None
        if k == 1:                                                          # gradients in another order than their parameters
            net.b.weight.grad = net.b.weight.grad.contiguous()
            net.a.weight.grad = net.a.weight.grad.to(memory_format=torch.channels_last)
        for a, b in zip(net.parameters(), ref.parameters()):
            b.grad = None if a.grad is None else a.grad.cpu().double()
        kept = [None if p.grad is None else p.grad.clone() for p in net.parameters()]
        own.step()
        norm = torch.nn.utils.clip_grad_norm_([p for p in ref.parameters() if p.grad is not None], 0.5)
        near_norm(own.grad_norm, float(norm))
        theirs.step()
        [r.step() for r in rates]
        close_steps(net.parameters(), ref.parameters(), 0.01, k + 1)
        assert all(a is None or torch.equal(a, p.grad) for a, p in zip(kept, net.parameters()))
    assert [float(own.state[p]["step"]) for p in net.parameters() if p in own.state] == [float(theirs.state[p]["step"]) for p in ref.parameters() if p in theirs.state]
    twin = Net().cuda()
    twin.load_state_dict(net.state_dict())
    again = optim.Adam(split(twin), max_grad_norm=0.5, ops=hip)
    again.load_state_dict(own.state_dict())
    for n in (net, twin):
        for p, q in zip(n.parameters(), net.parameters()):
            p.grad = None if q.grad is None else q.grad.clone()
    own.step()
    again.step()
    assert all(torch.equal(a, b) for a, b in zip(net.parameters(), twin.parameters()))


@gpu
def test_clip_grad_norm_of_a_module(hip):
    net = Net().cuda()
    net(torch.randn(2, 3, 16, 16).cuda()).square().mean().backward()
    had = [p.grad.cpu().double() for p in net.parameters() if p.grad is not None]
    norm = optim.clip_grad_norm(net.parameters(), 0.01)
    near_norm(norm, norm64(had))
    near_clipped([p.grad for p in net.parameters() if p.grad is not None], had, 0.01 / (norm64(had) + 1e-6))
    net.a.weight.grad[0] = math.nan
    with pytest.raises(RuntimeError):
        optim.clip_grad_norm(net.parameters(), 1.0, error_if_nonfinite=True)


@gpu
def test_captured_training_step(hip):
    """forward, backward, clip_grad_norm and the optimizer in one graph, against the same steps taken eagerly."""
    x = torch.randn(2, 3, 16, 16, generator=torch.Generator().manual_seed(9)).cuda()

    def steps(net, opt, n, x):
        for _ in range(n):
            opt.zero_grad()
            net(x).square().mean().backward()
            optim.clip_grad_norm(net.parameters(), 0.02, ops=hip)
            opt.step()

    eager, net = Net().cuda(), Net().cuda()
    lr = torch.tensor(0.01, device="cuda:0")
    opts = [optim.Adam(n.parameters(), lr=lr, ops=hip) for n in (eager, net)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        steps(net, opts[1], 2, x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    opts[1].zero_grad()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(net, opts[1], 1, x)
        fresh = optim.Adam(net.parameters(), ops=hip)
        with pytest.raises(RuntimeError):
            fresh.step()                                                    # would make its state at every replay
        assert not any(fresh.state[p] for p in net.parameters())
    steps(eager, opts[0], 2, x)
    for k in range(4):
        lr.fill_(0.01 / (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        steps(eager, opts[0], 1, x)
        torch.cuda.synchronize()
        # the convolutions' gradients are torch's; their order of sums may differ between the two, so an update may differ by a part of its own size
        for a, b in zip(net.parameters(), eager.parameters()):
            assert (a - b).abs().max() <= 2e-4 * (k + 3)
    assert [float(opts[1].state[p]["step"]) for p in net.parameters() if p.grad is not None] == [6.0] * 6


@gpu
def test_train_step_on_the_gpu(hip, golden_dir):
    """linf/train.py::train_step with the kernels' clipping and optimizer: gradients and the update follow from the unclipped run's."""
    import bfsr_amd.linf.train as train
    from test_linf_cpu import run_train_step_case
    plain, prior, _ = run_train_step_case(golden_dir, hip, device="cuda:0")
    grads = [p.grad.cpu().double() for p in prior.parameters()]
    norm = norm64(grads)
    share = norm / 2 / (norm + 1e-6)
    step = train.train_step
    try:
        train.train_step = lambda m, *a, **k: step(m, *a, **dict(k, max_grad_norm=norm / 2, optimizer=optim.Adam(m.parameters(), lr=0.01, ops=hip)))
        out, moved, _ = run_train_step_case(golden_dir, hip, device="cuda:0")
    finally:
        train.train_step = step
    assert abs(out["grad_norm"] - norm) <= 1e-5 * norm and out["loss"] == pytest.approx(plain["loss"], rel=1e-6)
    for a, g, b in zip(prior.parameters(), grads, moved.parameters()):
        assert (b.grad.cpu().double() - g * share).abs().max() <= 1e-4 * g.abs().max() + 1e-12
        first = 0.01 * (g * share) / ((g * share).abs() + 1e-8)                     # Adam's first step
        big = g.abs() > 1e-3 * g.abs().max()
        assert ((a.detach() - b.detach()).cpu().double() - first)[big].abs().max() <= 1e-5


@gpu
def test_versions_of_views_and_plain_tensors(hip):
    """In-place results count as changes of what they are seen through, once a call."""
    base = torch.ones(100, device="cuda:0")
    views, plain = [base[:10], base[20:50].view(5, 6)], torch.ones(7, device="cuda:0")
    leaf = torch.nn.Parameter(torch.ones(8, device="cuda:0"))
    before = base._version, plain._version, leaf._version
    hip.clip_grads(hip.tensor_list(views + [plain, leaf]), 0.5)
    assert (base._version, plain._version, leaf._version) == tuple(v + 1 for v in before) and views[1]._version == base._version
    with torch.enable_grad():
        y = (leaf * leaf).sum()
    zeros = [torch.zeros(8, device="cuda:0") for _ in range(2)]
    hip.adam([leaf], [torch.ones(8, device="cuda:0")], zeros[:1], zeros[1:], torch.zeros(1, device="cuda:0")).run(0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
