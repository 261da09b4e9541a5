"""The end of a training step in the calls around its kernels (ops.ListTable, bfsr_amd.optim): freed memory, captured graphs, checkpoints, groups, changing sets of gradients.

`host` runs the host side of the operators on CPU tensors: the table, the checks and the calls as they are, without the kernels."""
import contextlib
import ctypes as C
import gc
import math
import types

import pytest
import torch
from torch.multiprocessing.reductions import StorageWeakRef

from bfsr_amd import _lib, ops as O, optim

CPU = torch.device("cpu")
gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _grad():
    """Other test modules turn gradients off for the whole process."""
    with torch.enable_grad():
        yield


class Lib(object):
    """The C entries that a table needs, and a record of the calls."""

    def __init__(self):
        self.calls, self.gone, self.tickets = [], set(), 0

    def bfsr_list_chunk(self, total):
        return 2048

    def bfsr_list_work(self, n):
        return 2048 + 16 * n

    def bfsr_norm_work(self, count):
        return 0

    def bfsr_capture_ticket(self, stream, ticket):
        self.tickets += 1
        ticket._obj.value = self.tickets
        return 0

    def bfsr_capture_gone(self, ticket):
        return int(ticket in self.gone)

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return 0
        return entry


class Host(object):
    """An ops object whose launches are only recorded."""

    def __init__(self):
        self.lib, self.device, self._keylog, self.profile_keys = Lib(), CPU, None, None
        self.tensor_list, self.adam = (lambda *a, **k: self.made(O.TensorList(self, *a, **k))), (lambda *a: self.made(O.AdamPlan(self, *a)))
        self.plans = 0

    def made(self, table):
        self.plans += 1
        return table

    def _index_device(self):
        return CPU

    clip_grads, grad_norm, _listed, _norm_out = O.HipOps.clip_grads, O.HipOps.grad_norm, O.HipOps._listed, O.HipOps._norm_out


@pytest.fixture
def host(monkeypatch):
    stream = types.SimpleNamespace(cuda_stream=0, synchronize=lambda: None)
    ops = Host()
    ops.capturing = False
    for name, value in (("device", lambda d: contextlib.nullcontext()), ("is_current_stream_capturing", lambda: ops.capturing), ("current_stream", lambda d=None: stream),
                        ("current_device", lambda: None), ("synchronize", lambda d=None: None)):
        monkeypatch.setattr(torch.cuda, name, value)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: t.device.index, raising=False)       # None on the CPU, like the device's index
    monkeypatch.setattr(optim, "_ops_of", lambda t, ops_=None: ops_ or ops)
    monkeypatch.setattr(O, "_captured", type(O._captured)())
    yield ops


def make(shapes=((4,), (3, 5)), dtype=torch.float32):
    new = lambda: [torch.randn(s) for s in shapes]                  # noqa: E731
    return [t.to(dtype) for t in new()], [t.to(dtype) for t in new()], [t * 0 for t in new()], [t * 0 for t in new()], torch.zeros(len(shapes))


# ---- memory that is no longer there
def freed(shape=(4,), offset=0):
    """A tensor whose storage has been given back, as sharded training does between uses."""
    base = torch.ones(64)
    t = base[offset:offset + math.prod(shape)].view(shape)
    base.untyped_storage().resize_(0)
    return t


@pytest.mark.parametrize("offset", [0, 8])
def test_freed_storage_is_refused(host, offset):
    """Its address is an offset, which no kernel may follow."""
    t = freed(offset=offset)
    assert t.data_ptr() == 4 * offset
    with pytest.raises(ValueError, match="freed"):
        O._addresses([torch.ones(4), t])
    with pytest.raises(ValueError, match="freed"):
        host.tensor_list([t])
    with pytest.raises(ValueError, match="freed"):
        host.tensor_list([torch.ones(4)], out=[t])
    p, g, m, v, step = make(((4,),))
    for args in (([t], g, m, v, step), (p, [t], m, v, step), (p, g, [t], v, step), (p, g, m, [t], step), (p, g, m, v, [freed((), offset)])):
        with pytest.raises(ValueError, match="freed"):
            host.adam(*args)
    plan = host.adam(p, None, m, v, step)
    plan.run(0.1, grads=g)
    with pytest.raises(ValueError, match="freed"):
        plan.run(0.1, grads=[t])
    assert len([c for c in host.lib.calls if c[0] == "bfsr_adam_step"]) == 1
    w = torch.nn.Parameter(torch.ones(4))
    opt = optim.Adam([w], ops=host)
    w.grad = t
    with pytest.raises(ValueError, match="freed"):
        opt.step()
    O._addresses([torch.zeros(0), torch.zeros(3, 0)])               # nothing to be held
    shrunk = torch.ones(64)
    shrunk.untyped_storage().resize_(128)
    with pytest.raises(ValueError, match="freed"):
        O._held(shrunk, "x")
    O._held(shrunk[:32], "x")


# ---- gradients
def conjugated(values, device="cpu"):
    """A gradient of one element behind a lazy minus sign."""
    g = torch.complex(torch.zeros(1), -torch.tensor([values])).to(device).conj().imag
    assert g.is_neg() and float(g) == values
    return g


def test_lazily_negated_gradients_are_read(host):
    """A step without the gradients' addresses would take the parameters for them."""
    w = torch.nn.Parameter(torch.ones(1))
    opt = optim.Adam([w], ops=host)
    for _ in range(2):
        host.lib.calls.clear()
        w.grad = conjugated(0.25)
        opt.step()
        assert [c[0] for c in host.lib.calls if "write" in c[0] or "step" in c[0]][-2:] == ["bfsr_pointer_write", "bfsr_adam_step"]


def test_gradients_that_do_not_go_with_their_parameters_are_refused(host, monkeypatch):
    w = torch.nn.Parameter(torch.ones(1))
    w.grad = torch.ones(1)
    opt = optim.Adam([w], ops=host)
    monkeypatch.setattr(O.AdamPlan, "fit", lambda self, grads: None)
    with pytest.raises(ValueError):
        opt.step()


@gpu
def test_lazily_negated_gradients_on_the_gpu():
    got = []
    for lazy in (False, True):
        w = torch.nn.Parameter(torch.full((1,), 2.0, device="cuda:0"))
        opt = optim.Adam([w], lr=0.1)
        for g in (0.25, -0.5):
            w.grad = conjugated(g, "cuda:0") if lazy else torch.tensor([g], device="cuda:0")
            opt.step()
        got.append((float(w.detach()), float(opt.state[w]["exp_avg"])))
    assert got[0] == got[1] and got[0][1] == pytest.approx(0.9 * 0.025 - 0.05, abs=1e-8)


# ---- graphs: what a replay reads and writes lives as long as the graph
def refs(tensors):
    return [StorageWeakRef(t.untyped_storage()) for t in tensors]


def test_captured_calls_hold_their_memory(host):
    p, g, m, v, step = make()
    out = [torch.zeros_like(t) for t in g]
    lr, norm = torch.tensor(0.1), torch.tensor(2.0)
    plan, clip = host.adam(p, g, m, v, step), host.tensor_list(g, out=out)
    held = refs(p + m + v + g + [step, lr, norm])
    taken = refs(g + out)
    loose = refs(make()[0])
    host.capturing = True
    plan.run(lr, max_norm=1.0, grad_norm=norm)
    host.clip_grads(clip, 1.0)
    host.clip_grads([torch.ones(3)], 1.0)                           # a plain list's memory is the caller's to keep
    host.capturing = False
    del p, g, m, v, step, out, lr, norm, plan, clip
    gc.collect()
    host.tensor_list([torch.ones(3)])
    assert not any(r.expired() for r in held + taken) and all(r.expired() for r in loose) and len(O._captured) == 2
    host.lib.gone.add(1)
    host.tensor_list([torch.ones(3)])                               # the next table finds the first graph gone
    assert [r.expired() for r in held] == [True] * 6 + [False] * 2 + [True] * 3 and not any(r.expired() for r in taken)
    host.lib.gone.add(2)
    host.tensor_list([torch.ones(3)])
    assert all(r.expired() for r in held + taken) and not O._captured


def test_tickets_are_refused():
    lib = _lib.load()
    assert lib.bfsr_capture_ticket(None, None) == lib.bfsr_capture_gone(None) == -1


@gpu
def test_a_graph_outlives_its_plan():
    """Nothing else holds the captured plan's moments, counts and rate: replays still find them, memory that is taken meanwhile stays as it is, and it ends with the graph."""
    hip = O.HipOps("cuda:0")
    shapes = [(3000,), (17, 65), (70001,)]
    new = lambda f: [torch.full(s, f, device="cuda:0") for s in shapes]              # noqa: E731
    p, g, m, v, step = new(1.0), new(0.5), new(0.0), new(0.0), torch.zeros(3, device="cuda:0")
    lr = torch.tensor(0.25, device="cuda:0")
    plan = hip.adam(p, g, m, v, step)
    before = len(O._captured)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(lr, betas=(0.5, 0.5))
    ends = refs(m + v + [step, lr])
    del plan, m, v, step, lr
    gc.collect()
    junk = [new(7.0) for _ in range(4)] + [[torch.full((k,), 7.0, device="cuda:0") for k in (1, 1, 3, 3)]]
    hip.tensor_list(g)
    assert len(O._captured) == before + 1 and not any(r.expired() for r in ends)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        # a constant gradient: m / (1 - b^t) = g, v / (1 - b^t) = g^2, so each step takes lr away, but for a dozen roundings and eps
        for t in p:
            assert float((t - (0.75 - 0.25 * k)).abs().max()) <= 16 * 2.0 ** -24 * (k + 1) + 2e-8 * (k + 1)
    assert all(float(t.min()) == 7.0 == float(t.max()) for c in junk for t in c)
    del graph
    gc.collect()
    hip.tensor_list(g)
    assert len(O._captured) == before and all(r.expired() for r in ends)


# ---- checkpoints
@pytest.mark.parametrize("written", [True, False])
@pytest.mark.parametrize("theirs, decoupled", [(torch.optim.AdamW, True), (torch.optim.Adam, False)])
def test_decay_of_a_loaded_checkpoint(theirs, decoupled, written):
    """A checkpoint decides between the two decays where it says which one it used; older ones do not, and leave it to the optimizer that loads them."""
    w = [torch.nn.Parameter(torch.ones(3)) for _ in range(2)]
    saved = theirs([dict(params=[p], weight_decay=0.1 * (k + 1)) for k, p in enumerate(w)], lr=0.5).state_dict()
    for k, g in enumerate(saved["param_groups"]):
        g["decoupled_weight_decay"] = decoupled
        if not written:
            del g["decoupled_weight_decay"]
    opt = optim.Adam([dict(params=[w[0]], decoupled_weight_decay=True), dict(params=[w[1]], decoupled_weight_decay=False)], lr=0.1)
    opt.load_state_dict(saved)
    assert [g["decoupled_weight_decay"] for g in opt.param_groups] == ([decoupled] * 2 if written else [True, False])
    assert [(g["lr"], g["weight_decay"]) for g in opt.param_groups] == [(0.5, 0.1), (0.5, 0.2)]
    assert all(("decoupled_weight_decay" in g) == written for g in saved["param_groups"])              # the caller's dict stays as it was


def test_hooks_of_loading_see_to_moments_too():
    w = torch.nn.Parameter(torch.ones(3))
    saved = optim.Adam([w]).state_dict()
    saved["state"] = {0: {"step": torch.tensor(4.0), "exp_avg": torch.full((3,), 1.0), "exp_avg_sq": torch.full((3,), 2.0)}}
    opt = optim.Adam([w], lr=0.1)

    def twice(_, d):
        d["state"] = {0: {"step": torch.tensor(9.0), "exp_avg": d["state"][0]["exp_avg"] * 2, "exp_avg_sq": d["state"][0]["exp_avg_sq"] * 4}}
        d["param_groups"] = [dict(g, lr=0.7) for g in d["param_groups"]]
        return d

    hook = opt.register_load_state_dict_pre_hook(twice)
    for _ in range(2):
        opt.load_state_dict(saved)
        assert [float(opt.state[w][k].max()) for k in ("step", "exp_avg", "exp_avg_sq")] == [9.0, 2.0, 8.0] and opt.param_groups[0]["lr"] == 0.7
    hook.remove()
    opt.load_state_dict(saved)
    assert [float(opt.state[w][k].max()) for k in ("step", "exp_avg", "exp_avg_sq")] == [4.0, 1.0, 2.0] and opt.param_groups[0]["lr"] == 1e-3


@gpu
def test_a_graph_captured_before_a_checkpoint_is_loaded():
    """It goes on with the state that it was captured with, beside the new one."""
    hip = O.HipOps("cuda:0")
    w = [torch.nn.Parameter(torch.full((n,), 1.0, device="cuda:0")) for n in (5, 70001)]
    for p in w:
        p.grad = torch.full_like(p, 0.5)
    lr = torch.tensor(0.25, device="cuda:0")
    opt = optim.Adam(w, lr=lr, betas=(0.5, 0.5), ops=hip)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    ends = refs([t for p in w for t in opt.state[p].values()] + [lr])
    saved = {"state": {k: {"step": torch.tensor(7.0), "exp_avg": torch.zeros_like(p), "exp_avg_sq": torch.ones_like(p)} for k, p in enumerate(w)},
             "param_groups": [dict(opt.state_dict()["param_groups"][0], lr=torch.tensor(0.0, device="cuda:0"))]}
    del lr
    opt.load_state_dict(saved)
    opt.step()
    gc.collect()
    junk = [[torch.full_like(p, 7.0) for p in w] for _ in range(4)] + [[torch.full((2,), 7.0, device="cuda:0") for _ in range(4)]]
    assert not any(r.expired() for r in ends)
    state = [{k: t.clone() for k, t in opt.state[p].items()} for p in w]
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for p, s in zip(w, state):
            # steps of a constant gradient take the rate away: 0.25 by the ordinary step, none by the loaded rate of 0, 0.25 by each replay
            assert float((p.detach() - (0.5 - 0.25 * k)).abs().max()) <= (16 * 2.0 ** -24 + 2e-8) * (k + 2)
            assert all(torch.equal(t, opt.state[p][n]) for n, t in s.items()) and float(s["step"]) == 8.0
    assert all(float(t.min()) == 7.0 == float(t.max()) for c in junk for t in c)


# ---- norms that are not finite
BIG = 3.0e38                     # two of them: finite gradients of a norm that float32 does not hold


@gpu
@pytest.mark.parametrize("bad", [(BIG, BIG), (math.inf, 0.0), (0.0, -math.inf), (math.nan, 1.0), (1.0, math.nan)])
@pytest.mark.parametrize("size", [6, 70001])
@pytest.mark.parametrize("most", [None, 1.0])
def test_skipped_steps_do_not_depend_on_the_groups(size, bad, most):
    got = []
    for groups in (1, 2):
        torch.manual_seed(3)
        w = [torch.nn.Parameter(torch.randn(n, device="cuda:0")) for n in (size, 3, size)]
        opt = optim.Adam([dict(params=w)] if groups == 1 else [dict(params=w[:1]), dict(params=w[1:])], lr=0.01, weight_decay=0.1, max_grad_norm=most, skip_nonfinite=True)
        for p in w:
            p.grad = torch.randn_like(p)
        opt.step()
        had = [p.detach().clone() for p in w] + [t.clone() for p in w for t in opt.state[p].values()]
        w[0].grad[size // 2], w[2].grad[1] = bad
        opt.step()
        norm = float(opt.grad_norm)
        assert math.isnan(norm) if any(map(math.isnan, bad)) else norm == math.inf
        now = [p.detach() for p in w] + [t for p in w for t in opt.state[p].values()]
        assert all(torch.equal(a, b) for a, b in zip(had, now))
        w[0].grad[size // 2], w[2].grad[1] = 0.5, 0.25
        opt.step()
        assert math.isfinite(float(opt.grad_norm)) and all(float(opt.state[p]["step"]) == 2.0 for p in w)
        assert all(bool((p.detach() != b).any()) for p, b in zip(w, had))
        got.append([p.detach() for p in w])
    # the norm of two groups is rounded to float32 in between: a share off by 2^-24, and an update of at most 10 lr each that is off by a few of those
    assert all(float((a - b).abs().max()) <= 2 * 10 * 0.01 * 16 * 2.0 ** -24 + 2.0 ** -22 for a, b in zip(*got))


@gpu
@pytest.mark.parametrize("size", [6, 70001])
def test_norms_beyond_float32_are_infinite_everywhere(size):
    hip = O.HipOps("cuda:0")
    new = lambda: [torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda() for n in (size, 3)]               # noqa: E731
    g = new()
    g[0][size // 2] = g[1][1] = BIG
    assert float(hip.grad_norm(g)) == math.inf and float(hip.grad_norm(g, math.inf)) == torch.tensor(BIG).item()
    out = [torch.full_like(t, 9.0) for t in g]
    assert float(hip.clip_grads(hip.tensor_list(g, out=out), 1e38)) == math.inf and not any(bool(t.any()) for t in out)
    p, m, v, step = new(), [torch.zeros_like(t) for t in g], [torch.zeros_like(t) for t in g], torch.zeros(2, device="cuda:0")
    plan = hip.adam(p, g, m, v, step)
    assert float(plan.run(0.1, max_norm=1e38)) == math.inf                                    # a share of 0: the step is taken with gradients of 0
    assert all(torch.equal(a, b) for a, b in zip(p, new())) and not any(bool(t.any()) for t in m + v) and step.tolist() == [1.0, 1.0]
    for given in (math.inf, math.nan, -math.inf):
        assert not math.isfinite(float(plan.run(0.1, max_norm=1.0, grad_norm=torch.tensor(given, device="cuda:0"), skip_nonfinite=True)))
        assert step.tolist() == [1.0, 1.0] and all(torch.equal(a, b) for a, b in zip(p, new()))
    g[0][size // 2] = g[1][1] = 0.0
    assert float(plan.run(0.1, max_norm=1.0, grad_norm=torch.tensor(4.0, device="cuda:0"), skip_nonfinite=True)) == 4.0 and step.tolist() == [2.0, 2.0]
    g[0].fill_(0.0)
    g[0][0], g[1][:] = 3.4e38, 0.0                                                                # the largest that are held
    assert math.isfinite(float(hip.grad_norm(g))) and float(hip.clip_grads(g, 1.0)) == torch.tensor(3.4e38).item() and abs(float(g[0][0]) - 1.0) <= 2.0 ** -22


# ---- decoupled decay
@gpu
@pytest.mark.parametrize("lr, wd", [(1e-4, 1e-2), (1e-5, 1e-2), (1e-3, 0.1), (1e-2, 0.3)])
@pytest.mark.parametrize("size", [2000, 70001])
def test_small_decoupled_decay(size, lr, wd):
    """Without gradients a step is the decay alone: (lr wd) p, rounded as a number of its own (its factor, the product and the update: 3 u of it) and off the parameter (u of that).
    p times a rounded 1 - lr wd is off by up to half a u of p more, the same way for every p."""
    hip = O.HipOps("cuda:0")
    p = torch.randn(size, generator=torch.Generator().manual_seed(11)).cuda()
    zeros = [torch.zeros_like(p) for _ in range(3)]
    had, u = p.cpu().double(), 2.0 ** -24
    hip.adam([p], zeros[:1], zeros[1:2], zeros[2:], torch.zeros(1, device="cuda:0")).run(lr, weight_decay=wd, decoupled=True)
    want = had * (1 - lr * wd)
    assert bool(((p.cpu().double() - want).abs() <= want.abs() * u + had.abs() * lr * wd * 3 * u + 2.0 ** -149).all())


# ---- sets of parameters with gradients
def test_alternating_sets_keep_their_plans(host):
    """Conditional branches and partly frozen modules: each set's table is made once, and may be captured when it has been stepped with."""
    w = [torch.nn.Parameter(torch.ones(n)) for n in (3, 4, 5)]
    opt = optim.Adam([dict(params=w[:2]), dict(params=w[2:])], ops=host)

    def step(which):
        for k, p in enumerate(w):
            p.grad = torch.ones_like(p) if k in which else None
        opt.step()

    for _ in range(3):
        for which in ((0, 1, 2), (0,), (1, 2), (2,), ()):
            step(which)
    assert host.plans == 4                           # (0, 1), (0,) and (1,) of the first group, (2,) of the second
    host.capturing = True
    for which in ((0,), (1,), (0, 1, 2)):
        step(which)
    host.capturing = False
    assert host.plans == 4
    late = torch.nn.Parameter(torch.ones(2))
    opt.add_param_group(dict(params=[late]))
    late.grad = torch.ones(2)
    host.capturing = True
    with pytest.raises(RuntimeError):
        opt.step()
    host.capturing = False


def test_plans_of_other_memory_are_let_go(host):
    """A plan holds the parameters' and the state's memory: once they stand elsewhere it has to go, whichever set it was for."""
    w = [torch.nn.Parameter(torch.ones(n)) for n in (3, 4)]
    opt = optim.Adam(w, ops=host)

    def step(which):
        for k, p in enumerate(w):
            p.grad = torch.ones_like(p) if k in which else None
        opt.step()

    step((0, 1))
    step((0,))
    before = refs([w[0].detach()] + [opt.state[w[0]][k] for k in ("exp_avg", "exp_avg_sq")])
    w[0].data = torch.ones(3)
    for k in ("exp_avg", "exp_avg_sq"):
        opt.state[w[0]][k] = torch.zeros(3)
    assert not any(r.expired() for r in before)
    step((0,))
    gc.collect()
    assert all(r.expired() for r in before)
    made = host.plans
    step((0,))
    assert host.plans == made
    more = [torch.nn.Parameter(torch.ones(2)) for _ in range(4)]          # a few sets are remembered, not all
    opt = optim.Adam(more, ops=host)
    for bits in range(1, 16):
        for k, p in enumerate(more):
            p.grad = torch.ones_like(p) if bits >> k & 1 else None
        opt.step()
    assert len(opt._plans[0]) == optim.PLANS


@gpu
def test_alternating_sets_on_the_gpu():
    """Against torch's Adam in 64 bits, the sets in turn and from a graph of one of them."""
    hip = O.HipOps("cuda:0")
    values = [torch.randn(n, generator=torch.Generator().manual_seed(n)) for n in (3, 3001, 5)]
    own, ref = [torch.nn.Parameter(t.cuda()) for t in values], [torch.nn.Parameter(t.double()) for t in values]
    opt, theirs = optim.Adam(own, lr=0.01, ops=hip), torch.optim.Adam(ref, lr=0.01)
    static = [torch.zeros_like(p) for p in own]
    graph, taken = None, 0
    for k in range(8):
        which = ((0, 1, 2), (0,), (1, 2))[k % 3]
        for i, (a, b) in enumerate(zip(own, ref)):
            g = torch.randn(b.shape, generator=torch.Generator().manual_seed(10 * k + i))
            static[i].copy_(g)
            a.grad, b.grad = (static[i], g.double()) if i in which else (None, None)
        if k == 4:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        if graph is not None and k % 3 == 1:
            graph.replay()
        else:
            opt.step()
        theirs.step()
        taken += 1
        for a, b in zip(own, ref):
            # each step's update is at most about 10 lr and off by a few dozen roundings of itself, and two of the parameter
            assert bool(((a.detach().cpu().double() - b.detach()).abs() <= taken * 2.0 ** -24 * (4 * b.detach().abs() + 64 * 10 * 0.01)).all())
    assert [float(opt.state[p]["step"]) for p in own] == [float(theirs.state[p]["step"]) for p in ref] and len(opt._plans[0]) == 3


def test_a_parameter_turned_in_its_memory(host):
    """Same address, other order of the axes: the plan would pair its elements with others' gradients.  Its moments, in the old order, are refused; new ones go with it."""
    w = torch.nn.Parameter(torch.ones(3, 3))
    opt = optim.Adam([w], ops=host)
    w.grad = torch.ones(3, 3)
    opt.step()
    w.data = w.data.t()
    calls = len(host.lib.calls)
    with pytest.raises(ValueError, match="strides"):
        opt.step()
    assert not [c for c in host.lib.calls[calls:] if c[0] == "bfsr_adam_step"]
    opt.state.clear()
    opt.step()
    assert host.plans == 2 and opt.state[w]["exp_avg"].stride() == (1, 3)


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
def test_gradients_are_not_held(host, types):
    """zero_grad frees them, whatever their type."""
    w = torch.nn.Parameter(torch.ones(5, dtype=types[0]))
    w.grad_dtype = types[1]
    opt = optim.Adam([w], ops=host)
    for _ in range(2):
        w.grad = torch.ones(5, dtype=types[1])
        ends = refs([w.grad])
        opt.step()
        opt.zero_grad()
        gc.collect()
        assert ends[0].expired()
    assert host.plans == 1
    with pytest.raises(ValueError):
        opt._plans[0][0][2].run(0.1)                  # nor can the plan go by where they were


# ---- numbers on the device
@pytest.mark.parametrize("bad", [lambda: conjugated(0.5), lambda: torch.ones(1).to_sparse(), lambda: freed((1,)), lambda: freed((), 8)])
def test_numbers_on_the_device_are_real_memory(host, bad):
    """A lazy minus sign would be lost, a freed rate would count as 0 or be read at an offset, a freed `out` be written there."""
    p, g, m, v, step = make()
    plan = host.adam(p, g, m, v, step)
    t = bad()
    for call in (lambda: plan.run(t), lambda: plan.run(0.1, max_norm=1.0, grad_norm=t), lambda: host.grad_norm(g, out=t), lambda: host.grad_norm([], out=t),
                 lambda: host.adam(p[:1], g[:1], m[:1], v[:1], [t])):
        with pytest.raises(ValueError):
            call()
    assert not [c for c in host.lib.calls if c[0] in ("bfsr_adam_step", "bfsr_grad_norm")]
    plan.run(torch.tensor([0.5]), max_norm=1.0, grad_norm=torch.tensor(2.0))
    assert [c[0] for c in host.lib.calls][-1] == "bfsr_adam_step"


def test_a_norms_output_counts_as_changed(host):
    """A backward pass that needs what `out` held before has to say so."""
    g = make()[1]
    for tensors in (g, host.tensor_list(g), []):
        out = torch.ones(1)
        x = torch.ones(1, requires_grad=True)
        y = x * out
        version = out._version
        assert host.grad_norm(tensors, out=out) is out and out._version == version + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        host.grad_norm(g, out=torch.ones(()))


def test_bytes_of_a_list_with_an_output(host):
    """What a call touches decides whether it streams past the cache: a norm does not touch the output."""
    g = make()[1]
    total = sum(t.nbytes for t in g)
    for tensors, whole in ((host.tensor_list(g), total), (host.tensor_list(g, out=[torch.zeros_like(t) for t in g]), 2 * total)):
        host.grad_norm(tensors)
        host.clip_grads(tensors, 1.0)
        assert [args[0].bytes for name, args in host.lib.calls[-2:]] == [total, whole] and tensors.bytes == whole


def test_a_bound_that_is_no_number_is_refused():
    """... and not taken for `no clipping`, which any negative one is."""
    lib = _lib.load()
    a = _lib.BfsrListArgs(rows=4096, chunks=4096, n=1, count=1, chunk=lib.bfsr_list_chunk(1), work=4096, norm=4096)
    for skip in (0, 1):
        h = _lib.BfsrAdamArgs(beta1=0.9, beta2=0.999, max_norm=math.nan, skip_nonfinite=skip)
        assert lib.bfsr_adam_step(C.byref(a), C.byref(h), None) == -1 == lib.bfsr_clip_grads(C.byref(a), math.nan, None)


# ---- arguments of the optimizer
@pytest.mark.parametrize("bad", [dict(lr=torch.tensor(-0.1)), dict(lr=torch.tensor(math.nan)), dict(lr=torch.tensor([0.1, 0.1])), dict(lr=-1.0), dict(eps=math.nan), dict(betas=(0.9, 1.0)),
                                 dict(weight_decay=-1.0)])
def test_groups_out_of_range_are_refused(bad):
    w = [torch.nn.Parameter(torch.ones(3)) for _ in range(2)]
    for make_it in (lambda: optim.Adam(w, **bad), lambda: optim.Adam([dict(params=w[:1]), dict(params=w[1:], **bad)])):
        with pytest.raises(ValueError):
            make_it()
    opt = optim.Adam(w[:1], lr=torch.tensor(0.1))
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=w[1:], **bad))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=w[1:], lr=torch.tensor([0.0]), eps=0.5))
    assert [g["eps"] for g in opt.param_groups] == [1e-8, 0.5]


def test_the_norm_of_no_gradients_is_on_their_device():
    for w in (torch.nn.Parameter(torch.ones(3, device="meta")), [torch.nn.Parameter(torch.ones(3, device="meta"))], iter([torch.ones(3, device="meta")])):
        norm = optim.clip_grad_norm(w, 1.0)
        assert norm.device.type == "meta" and norm.shape == () and norm.dtype == torch.float32
    assert float(optim.clip_grad_norm([], 1.0)) == 0.0


def test_sparse_gradients_are_refused_at_every_step(host):
    w = torch.nn.Parameter(torch.ones(3))
    opt = optim.Adam([w], ops=host)
    for g in (torch.ones(3).to_sparse(), torch.ones(3), torch.ones(3).to_sparse(), torch.ones(3)):
        w.grad = g
        with pytest.raises(RuntimeError, match="sparse") if g.is_sparse else contextlib.nullcontext():
            opt.step()
    assert [c[0] for c in host.lib.calls].count("bfsr_adam_step") == 2


def test_captured_norms_hold_their_output(host):
    g, out = make()[1], torch.zeros(())
    tensors = host.tensor_list(g)
    ends = refs([out])
    host.capturing = True
    host.grad_norm(tensors, out=out)
    host.capturing = False
    del out
    gc.collect()
    assert not ends[0].expired()
    host.lib.gone.add(1)
    host.tensor_list(make()[1])
    assert ends[0].expired()


def test_numbers_that_the_update_writes_are_refused(host):
    """Some workgroups would read them before, some after."""
    p, g, m, v, step = make()
    plan = host.adam(p, g, m, v, step)
    for kw in [dict(lr=step[0])] + [dict(lr=0.1, max_norm=1.0, grad_norm=t) for t in (step[1], p[0][1], v[1][2, 1:2])]:
        with pytest.raises(ValueError, match="writes"):
            plan.run(**kw)
    plan.run(g[0][0], max_norm=1.0, grad_norm=g[1][0, 0])
    plan.run(p[0][0])                                               # a rate that is learned: read before the parameters are written


# ---- calls in other surroundings
@gpu
def test_captured_step_of_two_groups_with_a_common_norm():
    """Clipped by the norm over both groups, types mixed, against the same steps taken eagerly."""
    hip = O.HipOps("cuda:0")
    nets = []
    for _ in range(2):
        w = [torch.nn.Parameter(torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda().to(t)) for n, t in ((70001, torch.float32), (3, torch.bfloat16), (5000, torch.bfloat16))]
        w[2].grad_dtype = torch.float32
        opt = optim.Adam([dict(params=w[:1]), dict(params=w[1:], lr=0.1)], lr=0.01, weight_decay=0.1, max_grad_norm=1.0, skip_nonfinite=True, ops=hip)
        for p in w:
            p.grad = torch.zeros_like(p, dtype=p.grad_dtype or p.dtype)
        nets.append((w, opt))

    def fill(k):
        for w, _ in nets:
            for i, p in enumerate(w):
                p.grad.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * k + i)))

    side = torch.cuda.Stream()
    fill(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):                                   # ordinary steps on a stream of their own
        for _, opt in nets:
            opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nets[0][1].step()
    norm = nets[0][1].grad_norm
    for k in range(1, 5):
        fill(k)
        if k == 3:
            for w, _ in nets:
                w[1].grad[1] = math.inf
        graph.replay()
        nets[1][1].step()
        torch.cuda.synchronize()
        assert float(norm) == float(nets[1][1].grad_norm) and math.isinf(float(norm)) == (k == 3)
        for a, b in zip(nets[0][0], nets[1][0]):
            assert torch.equal(a.detach(), b.detach())
            assert all(torch.equal(nets[0][1].state[a][n], t) for n, t in nets[1][1].state[b].items())
    assert [float(nets[0][1].state[p]["step"]) for p in nets[0][0]] == [4.0] * 3


@gpu
@pytest.mark.parametrize("size", [5, 70001])
def test_a_learned_rate(size):
    """One of the parameters is the rate: read before it is written."""
    hip = O.HipOps("cuda:0")
    p, g = [torch.full((1,), 0.25, device="cuda:0"), torch.full((size,), 1.0, device="cuda:0")], [torch.ones(1, device="cuda:0"), torch.ones(size, device="cuda:0")]
    m, v, step = [torch.zeros_like(t) for t in p], [torch.zeros_like(t) for t in p], torch.zeros(2, device="cuda:0")
    hip.adam(p, g, m, v, step).run(p[0], betas=(0.5, 0.5))
    # the first step takes the rate away from all: within eps = 1e-8 of it, and a dozen roundings
    assert abs(float(p[0])) <= 1e-8 + 16 * 2.0 ** -24 and float((p[1] - 0.75).abs().max()) <= 1e-8 + 16 * 2.0 ** -24
