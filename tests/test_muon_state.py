"""Muon's state and arguments on the CPU: what it refuses before a kernel could run on it."""
import pytest
import torch


def make(*shapes, **kw):
    from turboadam_b200 import Muon

    params = [torch.nn.Parameter(torch.zeros(*s)) for s in shapes]
    return params, Muon(params, **kw)


def saved(*shapes):
    params, opt = make(*shapes)
    for p in params:
        opt.state[p]["momentum_buffer"] = torch.ones_like(p)
    return opt.state_dict()


def test_load_state_dict_refuses_a_momentum_of_another_shape():
    """Kernels write a momentum through its pointer, at the parameter's size."""
    params, opt = make((6, 8), (4, 5))
    opt.load_state_dict(saved((6, 8), (4, 5)))
    assert opt.state[params[1]]["momentum_buffer"].shape == (4, 5)
    for shapes in (((6, 8), (2, 3)), ((8, 6), (4, 5)), ((6, 8), (20,) * 2)):
        with pytest.raises(ValueError, match="momentum"):
            opt.load_state_dict(saved(*shapes))
        # and nothing has changed
        assert [tuple(opt.state[p]["momentum_buffer"].shape) for p in params] == [(6, 8), (4, 5)]


@pytest.mark.parametrize("bad", [torch.zeros(2, 3), torch.zeros(8, 6), torch.zeros(6, 8).double(),
                                 torch.zeros(6, 8, device="meta"), torch.zeros(48), "text"])
def test_step_refuses_a_momentum_that_does_not_fit(bad, monkeypatch):
    from turboadam_b200 import muon

    calls = []
    monkeypatch.setattr(muon, "run_ortho", lambda *a: calls.append(a))
    (p,), opt = make((6, 8))
    p.grad = torch.ones_like(p)
    opt.state[p]["momentum_buffer"] = bad
    with pytest.raises((ValueError, NotImplementedError, TypeError)):
        opt._step_device(opt.param_groups[0], p.device, [p])
    assert not calls
    opt.state[p]["momentum_buffer"] = torch.zeros(6, 8)
    opt._step_device(opt.param_groups[0], p.device, [p])
    assert len(calls) == 1


def test_step_refuses_a_gradient_of_another_shape(monkeypatch):
    """A parameter whose data was replaced keeps its old gradient."""
    from turboadam_b200 import muon

    calls = []
    monkeypatch.setattr(muon, "run_ortho", lambda *a: calls.append(a))
    (p,), opt = make((6, 8))
    p.grad = torch.ones_like(p)
    p.data = torch.zeros(16, 18)
    with pytest.raises(ValueError, match="gradient"):
        opt._step_device(opt.param_groups[0], p.device, [p])
    assert not calls


def test_step_raises_version_counters(monkeypatch):
    """The kernels write behind autograd's back; a backward pass through a graph that saved the
    parameter before the step has to notice, as with torch's own optimizers."""
    from turboadam_b200 import muon

    monkeypatch.setattr(muon, "run_ortho", lambda *a: None)
    (p, q), opt = make((6, 8), (4, 5))
    x = torch.ones(3, 8, requires_grad=True)
    loss = (x @ p.t()).sum()
    p.grad = torch.ones_like(p)
    opt._step_device(opt.param_groups[0], p.device, [p])
    m = opt.state[p]["momentum_buffer"]
    before = m._version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    opt._step_device(opt.param_groups[0], p.device, [p])
    assert m._version > before
    assert q._version == 0


BAD = [dict(lr=-1.0), dict(lr=float("nan")), dict(momentum=1.0), dict(momentum=-0.1),
       dict(weight_decay=-0.1), dict(adjust_lr_fn="match_rms"), dict(ns_steps=0), dict(eps=-1.0),
       dict(ns_coefficients=(1.0, 2.0))]


@pytest.mark.parametrize("bad", BAD)
def test_values_of_a_group_are_checked(bad):
    from turboadam_b200 import Muon

    p, q = (torch.nn.Parameter(torch.zeros(4, 5)) for _ in range(2))
    with pytest.raises(ValueError):
        Muon([dict(params=[p], **bad)])
    opt = Muon([p])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[q], **bad))
    assert [g["params"] for g in opt.param_groups] == [[p]]


def test_refused_group_is_not_added():
    from turboadam_b200 import Muon

    p, q = torch.nn.Parameter(torch.zeros(4, 5)), torch.nn.Parameter(torch.zeros(4))
    opt = Muon([p])
    with pytest.raises(ValueError, match="TurboAdam"):
        opt.add_param_group(dict(params=[q]))
    assert [g["params"] for g in opt.param_groups] == [[p]]
    opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2, 3))], lr=0.5,
                             adjust_lr_fn="match_rms_adamw"))
    assert [g["lr"] for g in opt.param_groups] == [1e-3, 0.5]


def test_unknown_adjustment_set_later_is_refused(monkeypatch):
    """A schedule or a loaded state may write into a group."""
    from turboadam_b200 import muon

    monkeypatch.setattr(muon, "run_ortho", lambda *a: None)
    (p,), opt = make((6, 8))
    p.grad = torch.ones_like(p)
    opt.param_groups[0]["adjust_lr_fn"] = "match_rms"
    with pytest.raises(ValueError, match="adjust_lr_fn"):
        opt._step_device(opt.param_groups[0], p.device, [p])


def test_copies_and_pickles_keep_the_momentum_dtype():
    """torch's optimizers carry defaults, state and groups over a deepcopy or a pickle only."""
    import copy
    import pickle

    (p,), opt = make((6, 8), lr=0.5, momentum_dtype=torch.bfloat16)
    opt.state[p]["momentum_buffer"] = torch.ones(6, 8, dtype=torch.bfloat16)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        q = other.param_groups[0]["params"][0]
        q.grad = torch.ones_like(q)
        assert other._fitting(q, q.device)[1].dtype == torch.bfloat16
        del other.state[q]["momentum_buffer"]
        assert other._fitting(q, q.device)[1].dtype == torch.bfloat16
        assert other.param_groups[0]["lr"] == 0.5
        other.load_state_dict(opt.state_dict())
        assert other.state[q]["momentum_buffer"].dtype == torch.bfloat16
