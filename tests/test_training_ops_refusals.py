"""What the C ABI of the norms and of AdamW's moments refuses, on the host, before anything is launched."""
import ctypes

import pytest
import torch

from crystalframer_amd import _lib, norms, optim

A = 4096          # an address that no refused call looks at


def _norm(**change):
    a = _lib.CfhResidualNorm()
    a.struct_size, a.rows, a.dim, a.x_stride, a.x, a.norm, a.eps = ctypes.sizeof(a), 4, 64, 64, A, 1, 1e-5
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(struct_size=8), b"struct_size"), (dict(dtype=3), b"dtype"), (dict(dtype=1, weight_dtype=2), b"weight_dtype"), (dict(norm=3), b"norm"),
    (dict(block_norm=-1), b"norm"), (dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"), (dict(dim=0), b"dim"), (dict(dim=16385), b"dim"),
    (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(gate_rows=3, gate=A, block=A), b"gate_rows"),
    (dict(gate_rows=1, block=A), b"gate_rows"), (dict(gate=A, block=A), b"gate_rows"), (dict(x=None), b"x must"), (dict(block_norm=1), b"block"),
    (dict(gate=A, gate_rows=1), b"block"), (dict(x_stride=-1), b"strides")])
def test_norm_arguments(change, word):
    lib, a = _lib.load(), _norm(**change)
    assert lib.cfh_residual_norm_forward(ctypes.byref(a), A, A, None, None) < 0 and word in lib.cfh_last_error()
    assert lib.cfh_residual_norm_backward_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.cfh_residual_norm_backward(ctypes.byref(a), A, A, A, A, None, None, None, None, None, None, A, 1 << 20, None) < 0


def test_norm_gradients_of_what_is_not_there():
    lib = _lib.load()
    a = _norm()
    need = lib.cfh_residual_norm_backward_workspace_bytes(ctypes.byref(a))
    assert need > 0
    call = lambda a, *outs, stats=A, ws=A, n=need: lib.cfh_residual_norm_backward(ctypes.byref(a), stats, A, A, *outs, ws, n, None)  # noqa: E731
    none = [None] * 7
    for k in (1, 2, 5, 6):
        assert call(a, *none[:k], A, *none[k + 1:]) < 0 and b"not there" in lib.cfh_last_error()
    assert call(a, *none, stats=None) < 0 and b"stats" in lib.cfh_last_error()
    assert call(a, *none, ws=None) < 0 and call(a, *none, n=need - 1) < 0 and call(a, *none, ws=A + 4) < 0
    assert b"workspace" in lib.cfh_last_error()
    b = _norm(block=A, block_stride=64, residual_scale=1.0, block_scale=0.5)
    assert call(b, A, A, *none[2:]) < 0 and b"differs" in lib.cfh_last_error()
    assert call(_norm(joined=1, block=A), *none) < 0 and b"joined" in lib.cfh_last_error()
    assert call(_norm(norm=0), *none) < 0 and b"gy" in lib.cfh_last_error()
    assert lib.cfh_residual_norm_forward(ctypes.byref(_norm(norm=0)), A, A, None, None) < 0
    assert lib.cfh_residual_norm_forward(ctypes.byref(_norm(joined=1)), A, A, None, None) < 0
    assert lib.cfh_residual_norm_forward(None, A, A, None, None) < 0


def _job(**change):
    jobs = (_lib.CfhParamJob * 1)()
    jobs[0].param, jobs[0].grad, jobs[0].n = A, A, 10
    for k, v in change.items():
        setattr(jobs[0], k, v)
    return jobs


def _state(**change):
    s = _lib.CfhMoments()
    s.exp_avg, s.exp_avg_sq, s.exp_avg_scale, s.exp_avg_sq_scale, s.size, s.bits = A, A, A, A, 128, 8
    for k, v in change.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("job,state,rates,word", [
    (dict(n=-1), {}, {}, b"n ="), (dict(n=(1 << 40) + 1), {}, {}, b"n ="), (dict(dtype=3), {}, {}, b"dtype"), (dict(param=None), {}, {}, b"NULL"),
    (dict(grad=None), {}, {}, b"NULL"), (dict(grad=A + 2), {}, {}, b"address"), (dict(dtype=1, param=A + 1), {}, {}, b"address"),
    (dict(first=32), {}, {}, b"elements"), (dict(first=-64), {}, {}, b"elements"), (dict(first=128), {}, {}, b"elements"),
    (dict(n=129), {}, {}, b"elements"), ({}, dict(bits=4), {}, b"bits"), ({}, dict(size=-1), {}, b"size"), ({}, dict(exp_avg=None), {}, b"NULL"),
    ({}, dict(exp_avg_scale=None), {}, b"NULL"), ({}, dict(exp_avg=A + 8), {}, b"aligned"), ({}, {}, dict(beta1=1.0), b"beta1"),
    ({}, {}, dict(beta2=-0.1), b"beta1"), ({}, {}, dict(eps=-1.0), b"eps"), ({}, {}, dict(step=None), b"step_dev"), ({}, {}, dict(scratch=None), b"scratch")])
def test_adamw_arguments(job, state, rates, word):
    lib = _lib.load()
    r = dict(beta1=0.9, beta2=0.99, eps=1e-8, step=A, scratch=A)
    r.update(rates)
    rc = lib.cfh_adamw_step_moments(_job(**job), 1, ctypes.byref(_state(**state)), 1e-3, r["beta1"], r["beta2"], r["eps"], 0.0, None, r["step"],
                                    r["scratch"], None)
    assert rc < 0 and word in lib.cfh_last_error()


def test_sums_of_squares_clipping_and_values_of_moments():
    lib = _lib.load()
    jobs = _job()
    need = lib.cfh_grad_square_sums_count(jobs, 1)
    assert need == 1 and lib.cfh_grad_square_sums_count(_job(n=0), 1) == 0 and lib.cfh_grad_square_sums_count(None, 0) == 0
    for args in ((None, 1, A, need), (jobs, -1, A, need), (jobs, 1, None, need), (jobs, 1, A, need - 1), (jobs, 1, A, need + 1), (jobs, 1, A + 4, need)):
        assert lib.cfh_grad_square_sums(*args, None) < 0
    assert lib.cfh_grad_square_sums_count(_job(dtype=7), 1) < 0
    for change in (dict(norm=None), dict(sums=None), dict(count=-1), dict(max_norm=-1.0), dict(max_norm=float("nan"))):
        clip = _lib.CfhGradClip()
        clip.sums, clip.count, clip.max_norm, clip.norm = A, 1, 1.0, A
        for k, v in change.items():
            setattr(clip, k, v)
        rc = lib.cfh_adamw_step_moments(jobs, 1, ctypes.byref(_state()), 1e-3, 0.9, 0.99, 1e-8, 0.0, ctypes.byref(clip), A, A, None)
        assert rc < 0 and b"clip" in lib.cfh_last_error()
    for state, m in ((_state(bits=32), A), (_state(exp_avg=None), A), (_state(), None)):
        assert lib.cfh_adamw_moments(ctypes.byref(state), m, A, None) < 0
    assert lib.cfh_adamw_moments(None, A, A, None) < 0


def test_structures_match_the_header():
    assert ctypes.sizeof(_lib.CfhResidualNorm) == 136 and ctypes.sizeof(_lib.CfhParamJob) == 40 and ctypes.sizeof(_lib.CfhMoments) == 48
    assert ctypes.sizeof(_lib.CfhGradClip) == 32


def test_python_refuses_host_tensors_and_wrong_options():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="HIP device"):
        norms.residual_norm(x)
    p = torch.nn.Parameter(torch.zeros(8))
    for bad in (dict(state_bits=16), dict(max_grad_norm=-1.0), dict(max_grad_norm=float("nan"))):
        with pytest.raises(ValueError):
            optim.AdamW([p], **bad)
    p.grad = torch.zeros(8)
    with pytest.raises(RuntimeError, match="HIP device"):
        optim.AdamW([p], state_bits=8).step()


@pytest.mark.parametrize("gate,rows", [((32,), 1), ((4, 6, 32), 24), ((4, 1, 32), 4), ((1, 1, 32), 1)])
def test_rows_of_a_gate(gate, rows):
    assert _lib.load_host().gate_rows(torch.zeros(gate), torch.zeros(4, 6, 32)) == rows


@pytest.mark.parametrize("gate", [(6, 32), (1, 6, 32), (4, 6, 1), (2, 1, 32), (31,), (4, 2, 32)])
def test_gates_that_do_not_fit(gate):
    with pytest.raises(ValueError):
        _lib.load_host().gate_rows(torch.zeros(gate), torch.zeros(4, 6, 32))
