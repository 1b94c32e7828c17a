"""AdamW and AdamW8bit on the GPU against plain forms on the CPU (64-bit, with
derived bounds; and fp32 numpy, bit for bit), over types, sizes, layouts and
values where the kernels can go wrong."""

import copy

import numpy as np
import pytest
import torch

from _adamw_ref import EPS32, Plain32, Plain64, decode, encode
from smo_optimizer_b200 import SMO8bit, AdamW, AdamW8bit, _lib, clip_grad_norm_, grad_norm
from smo_optimizer_b200.zero import Zero1

pytestmark = pytest.mark.gpu

HP = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
ARGS = (HP["lr"], HP["betas"], HP["eps"], HP["weight_decay"])
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one element, around a lane's eight, blocks of 64 to 256, a chunk of 2048, several chunks
SIZES = [1, 7, 8, 9, 63, 64, 65, 127, 129, 255, 256, 257, 2047, 2048, 2049, 4101, 20003]


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")


def _np(t):
    return t.detach().float().cpu().numpy().reshape(-1)


def _rounder(dtype):
    if dtype == torch.float32:
        return None
    return lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dtype).to(
        torch.float64 if x.dtype == np.float64 else torch.float32).numpy()


def _rng(seed):
    return np.random.default_rng(seed)


def _params(sizes, dtype, seed=0, scale=0.1):
    r = _rng(seed)
    return [torch.nn.Parameter(torch.from_numpy(r.normal(0, scale, n).astype(np.float32)).cuda().to(dtype))
            for n in sizes]


def _grads(params, seed, scale=1e-2):
    r = _rng(seed)
    for p in params:
        p.grad = torch.from_numpy(r.normal(0, scale, tuple(p.shape)).astype(np.float32)).cuda().to(p.dtype)


def _same(a, b, what):
    """equal bits, with NaN equal to NaN"""
    a, b = np.asarray(a), np.asarray(b)
    assert a.shape == b.shape, what
    ok = (a == b) | (np.isnan(a) & np.isnan(b)) if a.dtype.kind == "f" else a == b
    assert ok.all(), f"{what}: {np.flatnonzero(~ok.reshape(-1))[:8]} of {ok.size}"


def _check_param(got, ref, what):
    """The parameter's bits with fp32 moments; within tol_p with 8-bit moments."""
    if not ref.block:
        return _same(got, ref.p, what)
    with np.errstate(invalid="ignore"):
        ok = (got == ref.p) | (np.isnan(got) & np.isnan(ref.p)) | (np.abs(got.astype(np.float64) - ref.p) <= ref.tol_p)
    assert ok.all(), f"{what}: {np.flatnonzero(~ok)[:8]} of {ok.size}"


def _check_codes(state, ref, what):
    for k, (c, s) in zip("mv", ref.codes):
        _same(state[k + "_q"].cpu().numpy().astype(np.int32), c, f"{what}: {k}_q")
        _same(state[k + "_s"].cpu().numpy(), s, f"{what}: {k}_s")


# ---------------------------------------------------------------- against 64 bits


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_adamw_against_64_bits(dtype, master):
    if master and dtype == torch.float32:
        pytest.skip("fp32 parameters have no master copy")
    params = _params(SIZES, dtype)
    opt = AdamW(params, master_weights=master, **HP)
    # a step of a type is eps relative to the value; a master copy is fp32
    direct = None if master else _rounder(dtype)
    info = torch.finfo(dtype)
    spacing = (0.0, 0.0) if direct is None else (info.eps, info.eps * info.smallest_normal)
    refs = [Plain64(_np(p), direct, *spacing) for p in params]
    for step in range(3):
        _grads(params, 10 + step)
        for p, r in zip(params, refs):
            r.step(_np(p.grad), *ARGS)
        opt.step()
    for p, r, n in zip(params, refs, SIZES):
        st = opt.state[p]
        assert st["step"] == 3 and st["exp_avg"].dtype == torch.float32
        assert (np.abs(_np(st["exp_avg"]) - r.m) <= r.tol_m).all(), n
        assert (np.abs(_np(st["exp_avg_sq"]) - r.v) <= r.tol_v).all(), n
        held = st["master"] if master else p
        assert (np.abs(_np(held) - r.p) <= r.tol_p).all(), n
        if master:
            assert torch.equal(p.detach(), st["master"].to(dtype)), n


@pytest.mark.parametrize("block", [64, 128, 256])
def test_adamw8_moments_are_within_half_a_code(block):
    """Each step's moments, as coded, against the 64-bit step from the same coded moments."""
    n = 5 * 256 + 77
    params = _params([n], torch.float32)
    p = params[0]
    opt = AdamW8bit(params, block_size=block, min_8bit_numel=0, **HP)
    b1, b2 = HP["betas"]
    m0 = v0 = np.zeros(n)
    for step in range(4):
        _grads(params, 30 + step)
        g = _np(p.grad).astype(np.float64)
        opt.step()
        m1, v1 = [_np(t).astype(np.float64) for t in opt.moments(p)[0]]
        m, u = b1 * m0 + (1 - b1) * g, np.sqrt(b2 * v0 + (1 - b2) * g * g)
        st = opt.state[p]
        for got, want, key, top in ((m1, m, "m", 127), (np.sqrt(v1), u, "v", 255)):
            c = np.abs(st[key + "_q"].cpu().numpy().astype(np.float64).reshape(-1)[:n])
            s = np.repeat(_np(st[key + "_s"]).astype(np.float64), block)[:n]
            # rounding to code c covers (c - 1/2)^2 .. (c + 1/2)^2 steps: (c + 1/4) / top^2 of s around c^2; a root
            # that would be 0 is lifted to 1; twelve fp32 roundings on the way, relative to s
            half = (c + 0.25) / top ** 2 + (c == 1) / top ** 2
            assert (np.abs(got - want) <= s * (half + 12 * EPS32)).all(), (key, step)
        m0, v0 = m1, v1


# ---------------------------------------------------------------- bit for bit


@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("block", [None, 64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_step_gives_the_definitions_bits(dtype, block, clip):
    params = _params(SIZES, dtype)
    kw = dict(HP, max_grad_norm=0.25 if clip else None)
    opt = AdamW(params, **kw) if block is None else AdamW8bit(params, block_size=block, min_8bit_numel=0, **kw)
    refs = [Plain32(_np(p), block, _rounder(dtype)) for p in params]
    for step in range(4):
        _grads(params, 50 + step)
        c = None
        if clip:
            total = np.float32(np.sqrt(sum(np.square(_np(p.grad).astype(np.float64)).sum() for p in params)))
            c = min(np.float32(1), np.float32(0.25) / (total + np.float32(1e-6)))
            assert c < 1
        kept = [p.grad.clone() for p in params]
        opt.step()
        for p, r, g in zip(params, refs, kept):
            r.step(_np(g), *ARGS, scale=c)
            assert torch.equal(p.grad, g)  # the gradients stay
        if clip:
            assert float(opt.last_grad_norm) == total
    for p, r, n in zip(params, refs, SIZES):
        _check_param(_np(p), r, n)
        if block is None:
            _same(_np(opt.state[p]["exp_avg"]), r.m, n)
            _same(_np(opt.state[p]["exp_avg_sq"]), r.v, n)
        else:
            _check_codes(opt.state[p], r, n)


@pytest.mark.parametrize("block", [None, 128])
@pytest.mark.parametrize("kind", ["zero", "tiny", "huge", "inf", "nan", "mixed"])
def test_odd_values(kind, block):
    """Zeros, values whose squares under- or overflow, infinities and NaN, in some of the blocks."""
    n = 128 * 6 + 5
    params = _params([n], torch.float32)
    p = params[0]
    opt = AdamW(params, **HP) if block is None else AdamW8bit(params, block_size=block, min_8bit_numel=0, **HP)
    ref = Plain32(_np(p), block)
    r = _rng(3)
    for step in range(3):
        g = r.normal(0, 1e-2, n).astype(np.float32)
        part = slice(130, 300)
        if kind == "zero":
            g[part] = 0.0
            g[-3:] = -0.0
        elif kind == "tiny":
            g[part] *= np.float32(1e-28)
            g[300:310] = np.float32(1e-43)
        elif kind == "huge":
            g[part] *= np.float32(1e24)
        elif kind == "inf":
            g[200] = np.inf
            g[400] = -np.inf
        elif kind == "nan":
            g[200] = np.nan
            g[-1] = np.nan
        else:
            g = (g * 10.0 ** r.uniform(-30, 10, n)).astype(np.float32)
        p.grad = torch.from_numpy(g).cuda()
        opt.step()
        ref.step(g, *ARGS)
        _check_param(_np(p), ref, (kind, step))
        if block:
            _check_codes(opt.state[p], ref, (kind, step))
        else:
            _same(_np(opt.state[p]["exp_avg"]), ref.m, (kind, step))
            _same(_np(opt.state[p]["exp_avg_sq"]), ref.v, (kind, step))


def _flat_views(sizes, dtype, lead):
    """Parameters and gradients as neighbouring views of two flat buffers, the first ``lead`` elements in."""
    total = lead + sum(sizes)
    r = _rng(8)
    flat, gflat = (torch.from_numpy(r.normal(0, s, total).astype(np.float32)).cuda().to(dtype) for s in (0.1, 0.01))
    params, o = [], lead
    for n in sizes:
        p = torch.nn.Parameter(flat[o:o + n])
        p.grad = gflat[o:o + n]
        params.append(p)
        o += n
    return flat, params


@pytest.mark.parametrize("block", [None, 64])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead", [1, 2, 3, 4, 8])
def test_unaligned_views_touch_only_their_elements(lead, dtype, block):
    sizes = [5, 2051, 1, 130, 4096, 700]
    flat, params = _flat_views(sizes, dtype, lead)
    before = flat[:lead].clone()
    opt = AdamW(params, **HP) if block is None else AdamW8bit(params, block_size=block, min_8bit_numel=0, **HP)
    refs = [Plain32(_np(p), block, _rounder(dtype)) for p in params]
    for _ in range(2):
        opt.step()
        for p, r in zip(params, refs):
            r.step(_np(p.grad), *ARGS)
    assert torch.equal(flat[:lead], before)
    for p, r in zip(params, refs):
        _check_param(_np(p), r, (lead, p.numel()))
        if block:
            _check_codes(opt.state[p], r, (lead, p.numel()))


@pytest.mark.parametrize("block", [None, 128])
def test_strided_parameters_and_gradients(block):
    """Transposed, sliced and channels-last parameters, and expanded gradients, against contiguous ones."""
    base = torch.from_numpy(_rng(4).normal(0, 0.1, (96, 80)).astype(np.float32)).cuda()
    conv = torch.from_numpy(_rng(5).normal(0, 0.1, (8, 6, 4, 4)).astype(np.float32)).cuda()
    strided = [base.clone().t(), base.clone()[:, 3:40], conv.clone().to(memory_format=torch.channels_last),
               base.clone()]
    params = [torch.nn.Parameter(t) for t in strided]
    plain = [torch.nn.Parameter(t.detach().contiguous().clone()) for t in strided]
    kw = dict(HP, max_grad_norm=0.5)
    cls, more = (AdamW, {}) if block is None else (AdamW8bit, dict(block_size=block, min_8bit_numel=0))
    a, b = cls(params, **more, **kw), cls(plain, **more, **kw)
    for step in range(3):
        for i, (p, q) in enumerate(zip(params, plain)):
            g = torch.from_numpy(_rng(60 + 10 * step + i).normal(0, 1e-2, tuple(p.shape)).astype(np.float32)).cuda()
            q.grad = g
            p.grad = g[:, :1].expand(96, 80) if i == 3 else g
            if i == 3:
                q.grad = p.grad.contiguous()
        a.step()
        b.step()
        for p, q in zip(params, plain):
            assert torch.equal(p.detach(), q.detach())
            assert a.state[p]["step"] == step + 1
            for k in b.state[q]:
                if torch.is_tensor(b.state[q][k]):
                    assert torch.equal(a.state[p][k], b.state[q][k]), k
    assert params[0].stride() == (1, 80)


@pytest.mark.parametrize("block", [None, 128])
def test_many_tensors_types_groups_and_missing_gradients(block):
    """More tensors than a launch holds, more scalars than a launch holds, all types at once, some without gradients
    or without elements."""
    r = _rng(11)
    sizes = [int(x) for x in r.integers(1, 400, 700)]
    params = []
    for i, n in enumerate(sizes):
        params += _params([n], TYPES[i % 3], seed=i)
    params += [torch.nn.Parameter(torch.zeros(0, device="cuda")), torch.nn.Parameter(torch.zeros(0, 5, device="cuda"))]
    groups = [{"params": params[i::40], "lr": 1e-3 * (1 + i)} for i in range(40)]
    opt = AdamW(groups, **HP) if block is None else AdamW8bit(groups, block_size=block, min_8bit_numel=100, **HP)
    refs = [Plain32(_np(p), block if block and p.numel() >= 100 else None, _rounder(p.dtype)) for p in params]
    steps = [0] * len(params)
    for step in range(3):
        _grads(params, 100 + step)
        for i, p in enumerate(params):
            if (i + step) % 5 == 0:
                p.grad = None
            else:
                steps[i] += 1
                refs[i].step(_np(p.grad), 1e-3 * (1 + i % 40), *ARGS[1:])
        opt.step()
    for i, (p, ref) in enumerate(zip(params, refs)):
        if steps[i]:
            assert opt.state[p]["step"] == steps[i]
            assert ("m_q" in opt.state[p]) == bool(ref.block)
        _check_param(_np(p), ref, (i, p.numel()))


@pytest.mark.parametrize("block", [None, 256])
def test_host_path_and_python_path_give_the_same_bits(block):
    sizes = [300, 5000, 17, 4096]

    def make():
        params = _params(sizes, torch.bfloat16)
        kw = dict(HP, master_weights=True, max_grad_norm=0.1)
        return params, AdamW(params, **kw) if block is None else AdamW8bit(params, block_size=block, **kw)

    (pa, a), (pb, b) = make(), make()
    for step in range(4):
        _grads(pa, 70 + step)
        _grads(pb, 70 + step)
        if step == 2:
            for o in (a, b):
                o.param_groups[0]["lr"] = 5e-3
        a.step()
        b._slow_step(b._ready(), None)
    assert a._plan is not None and b._plan is None
    assert torch.equal(a.last_grad_norm, b.last_grad_norm)
    for p, q in zip(pa, pb):
        assert torch.equal(p.detach(), q.detach())
        assert a.state[p].keys() == b.state[q].keys() and a.state[p]["step"] == b.state[q]["step"] == 4
        for k, t in a.state[p].items():
            assert not torch.is_tensor(t) or torch.equal(t, b.state[q][k]), k


def test_plan_follows_replaced_tensors():
    """New gradients, parameters, state tensors, groups and hyperparameters between two steps are all seen."""
    params = _params([500, 6000], torch.float32)
    opt = AdamW8bit(params, **HP)
    refs = [Plain32(_np(params[0])), Plain32(_np(params[1]), 128)]

    def both(lr=HP["lr"]):
        _grads(params, 7)
        opt.step()
        for p, r in zip(params, refs):
            r.step(_np(p.grad), lr, *ARGS[1:])

    both()
    params[0].data = params[0].data.clone()
    both()
    opt.state[params[0]]["exp_avg"] = opt.state[params[0]]["exp_avg"].clone()
    opt.state[params[1]]["m_s"] = opt.state[params[1]]["m_s"].clone()
    both()
    opt.param_groups[0]["lr"] = 3e-3
    both(3e-3)
    extra = _params([900], torch.float32, seed=5)
    opt.add_param_group({"params": extra, "lr": 3e-3})
    params.append(extra[0])
    refs.append(Plain32(_np(extra[0])))
    both(3e-3)
    opt.param_groups = [dict(g) for g in opt.param_groups]
    opt.param_groups[0]["lr"] = opt.param_groups[1]["lr"] = 2e-3
    both(2e-3)
    state = type(opt.state)(dict)
    for p, st in opt.state.items():
        state[p] = {k: (t.clone() if torch.is_tensor(t) else t) for k, t in st.items()}
    old, opt.state = opt.state, state
    both(2e-3)
    assert old[params[0]]["step"] + 1 == state[params[0]]["step"]
    for p, r in zip(params, refs):
        _check_param(_np(p), r, p.numel())


# ---------------------------------------------------------------- scaling


def test_grad_scale_and_clipping_together():
    params = _params([3000, 40], torch.float32)
    opt = AdamW(params, max_grad_norm=0.25, **HP)
    scale = torch.tensor(2.0 ** -3, device="cuda")
    _grads(params, 1, scale=10.0)
    refs = [Plain32(_np(p)) for p in params]
    total = np.float32(np.sqrt(sum(np.square(_np(p.grad).astype(np.float64)).sum() for p in params)) / 8)
    opt.step(grad_scale=scale)
    assert float(opt.last_grad_norm) == total
    c = np.float32(0.25) / (total + np.float32(1e-6)) * np.float32(0.125)
    for p, r in zip(params, refs):
        r.step(_np(p.grad), *ARGS, scale=c)
        _check_param(_np(p), r, p.numel())
    with pytest.raises(TypeError):
        opt.step(grad_scale=0.5)
    with pytest.raises(TypeError):
        opt.step(grad_scale=torch.ones(2, device="cuda"))
    with pytest.raises(RuntimeError):
        opt.step(grad_scale=torch.ones(()))
    assert opt.state[params[0]]["step"] == 1  # a refused step counts nothing


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_norm_clip_and_step_as_one_run(cls):
    """grad_norm, clip_grad_norm_ and a plain step give the bits of a step that clips by itself; the clipped
    gradients then go through SMO8bit too."""
    a, b = _params(SIZES, torch.float32), _params(SIZES, torch.float32)
    oa, ob = cls(a, max_grad_norm=0.25, **HP), cls(b, **HP)
    for step in range(3):
        _grads(a, 90 + step)
        _grads(b, 90 + step)
        oa.step()
        norm = grad_norm(b)
        assert torch.equal(clip_grad_norm_(b, 0.25), norm) and torch.equal(norm, oa.last_grad_norm)
        ob.step()
        assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(a, b))
    assert float(grad_norm(b)) == pytest.approx(0.25, rel=1e-4)
    smo = SMO8bit(b, lr=1e-3)
    smo.step()
    assert all(torch.isfinite(p).all() for p in b)


# ---------------------------------------------------------------- state


@pytest.mark.parametrize("block", [64, 128, 256])
def test_codes_to_numbers_and_back(block):
    n = 128 * 9 + 3
    r = _rng(21)
    m, u = (r.normal(0, 1, n) * 10.0 ** r.uniform(-6, 0, n)).astype(np.float32), None
    u = np.abs(m[::-1]).copy()
    u[5:90] = 0.0
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    wide, eight = AdamW([p], **HP), AdamW8bit([p], block_size=block, min_8bit_numel=0, **HP)
    wide.state[p] = {"step": 7, "exp_avg": torch.from_numpy(m).cuda(), "exp_avg_sq": torch.from_numpy(u).cuda().square()}
    root = np.sqrt(u * u)
    eight.load_state_dict(wide.state_dict())
    st = eight.state[p]
    assert st["step"] == 7 and set(st) == {"step", "m_q", "m_s", "v_q", "v_s"}
    (cm, sm), (cu, su) = encode(m, 127, block), encode(root, 255, block)
    _same(st["m_q"].cpu().numpy().astype(np.int32), cm, "m_q")
    _same(st["v_q"].cpu().numpy().astype(np.int32), cu, "v_q")
    dm, du = decode(cm, sm, 127).reshape(-1)[:n], decode(cu, su, 255).reshape(-1)[:n]
    out = (torch.full((n,), -1.0, device="cuda"), torch.full((n,), -1.0, device="cuda"))
    assert eight.moments([p], out=[out])[0] is out
    for got in (out, eight.moments()[0]):
        _same(_np(got[0]), dm, "m")
        _same(_np(got[1]), du * du, "v")
    back = AdamW([p], **HP)
    back.load_state_dict(eight.state_dict())
    _same(_np(back.state[p]["exp_avg"]), dm, "m")
    _same(_np(back.state[p]["exp_avg_sq"]), du * du, "v")


def test_moments_of_mixed_sets_and_refusals():
    params = _params([5000, 30], torch.float32)
    opt = AdamW8bit(params, **HP)
    _grads(params, 2)
    opt.step()
    pairs = opt.moments()
    assert pairs[1][0] is opt.state[params[1]]["exp_avg"]
    out = [tuple(torch.empty_like(p) for _ in range(2)) for p in params]
    opt.moments(params, out=out)
    for a, b in zip(pairs, out):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # views at odd addresses
    flat = torch.zeros(2, 5001, device="cuda")
    odd = (flat[0, 1:], flat[1, 1:])
    opt.moments(params[0], out=[odd])
    assert torch.equal(odd[0], out[0][0]) and torch.equal(odd[1], out[0][1]) and float(flat[0, 0]) == 0.0
    with pytest.raises(ValueError):
        opt.moments(params, out=out[:1])
    with pytest.raises(TypeError):
        opt.moments(params[0], out=[(torch.empty(5000, device="cuda"), torch.empty(5000, device="cuda").half())])
    with pytest.raises(TypeError):
        opt.moments(params[0], out=[(torch.empty(5000), torch.empty(5000))])
    with pytest.raises(KeyError):
        opt.moments(_params([10], torch.float32))


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_state_dict_continues_with_the_same_bits(cls):
    def make():
        params = _params([5000, 30, 257], torch.bfloat16)
        return params, cls(params, master_weights=True, **HP)

    pa, a = make()
    for step in range(2):
        _grads(pa, step)
        a.step()
    pb, b = make()
    with torch.no_grad():
        for p, q in zip(pa, pb):
            q.copy_(p)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    c = copy.deepcopy(a)  # parameters and all
    pc = c.param_groups[0]["params"]
    for p, q in zip(pa, pb):
        for k, t in a.state[p].items():
            assert not torch.is_tensor(t) or (t.dtype == b.state[q][k].dtype and torch.equal(t, b.state[q][k])), k
    for params, o in ((pa, a), (pb, b), (pc, c)):
        _grads(params, 9)
        o.step()
    for p, q, s in zip(pa, pb, pc):
        assert torch.equal(p.detach(), q.detach()) and torch.equal(p.detach(), s.detach())
        assert torch.equal(a.state[p]["master"], b.state[q]["master"])


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_loaded_states_share_nothing(cls, capturable):
    pa, pb = _params([5000, 30], torch.bfloat16), _params([5000, 30], torch.bfloat16)
    kw = dict(HP, master_weights=True, capturable=capturable, max_grad_norm=0.5)
    a, b = cls(pa, **kw), cls(pb, **kw)
    _grads(pa, 1)
    a.step()
    b.load_state_dict(a.state_dict())
    kept = copy.deepcopy(a.state_dict())
    for step in range(2):
        _grads(pb, 2 + step)
        b.step()
    for p, (i, st) in zip(pa, kept["state"].items()):
        for k, t in st.items():
            now = a.state[p][k]
            assert torch.equal(now, t) if torch.is_tensor(t) else now == t, k
    assert float(b.state[pb[0]]["step"]) == 3


def test_loads_a_torch_adamw_state():
    params = _params([5000, 30], torch.float32)
    ref = torch.optim.AdamW(params, **HP)
    _grads(params, 1)
    ref.step()
    wide, eight = AdamW(params, **HP), AdamW8bit(params, **HP)
    for opt in (wide, eight):
        opt.load_state_dict(ref.state_dict())
        assert opt.state[params[0]]["step"] == 1 and "block_size" in opt.param_groups[0] or opt is wide
        opt.step()
        assert opt.state[params[1]]["step"] == 2
    assert "m_q" in eight.state[params[0]] and "exp_avg" in eight.state[params[1]]


def test_bad_states_are_refused():
    params = _params([5000], torch.float32)
    opt = AdamW8bit(params, **HP)
    _grads(params, 1)
    opt.step()
    good = copy.deepcopy(opt.state_dict())
    bad = copy.deepcopy(good)
    bad["state"][0]["m_q"] = bad["state"][0]["m_q"][:-1]
    with pytest.raises(ValueError):
        opt.load_state_dict(bad)
    opt.load_state_dict(good)
    st = opt.state[params[0]]
    keep = st["m_q"]
    st["m_q"] = keep.float()
    with pytest.raises(TypeError):
        opt.step()
    st["m_q"] = keep[:-1]
    with pytest.raises(ValueError):
        opt.step()
    st["m_q"] = keep
    opt.step()
    assert st["step"] == 2


# ---------------------------------------------------------------- streams, devices, sizes


def test_runs_on_the_current_stream():
    params = _params([100_000], torch.float32)
    opt = AdamW8bit(params, **HP)
    ref = Plain32(_np(params[0]), 128)
    side = torch.cuda.Stream()
    _grads(params, 3)
    g = _np(params[0].grad)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        params[0].grad.mul_(2.0)
        for _ in range(3):
            opt.step()
            ref.step(2 * g, *ARGS)
        assert float(grad_norm(params)) == pytest.approx(float(np.linalg.norm(2.0 * g.astype(np.float64))), rel=1e-6)
    side.synchronize()
    _check_param(_np(params[0]), ref, "side stream")


def test_more_than_2_to_31_elements():
    n = 2 ** 31 + 4096 + 13
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros_like(p)
    tail = torch.from_numpy(_rng(1).normal(0, 1e-2, 5000).astype(np.float32)).bfloat16()
    p.grad[-5000:] = tail.cuda()
    opt = AdamW8bit([p], max_grad_norm=1e6, **HP)
    opt.step()
    first = n - 5000 - (n - 5000) % 128  # a block's begin before the tail
    g = np.zeros(n - first, np.float32)
    g[-5000:] = _np(tail)
    ref = Plain32(np.zeros(n - first), 128, _rounder(torch.bfloat16))
    ref.step(g, *ARGS)
    _check_param(_np(p[first:]), ref, "tail")
    for k, (c, s) in zip("mv", ref.codes):
        _same(opt.state[p][k + "_q"][first // 128:].cpu().numpy().astype(np.int32), c, k)
        _same(opt.state[p][k + "_s"][first // 128:].cpu().numpy(), s, k)
    assert float(opt.last_grad_norm) == np.float32(np.linalg.norm(g.astype(np.float64)))
    assert not p[:1 << 20].any() and not opt.state[p]["m_q"][: 1 << 20].any()


def test_zero1_on_one_rank_steps_adamw():
    a, b = _params([5000, 30], torch.bfloat16), _params([5000, 30], torch.bfloat16)
    kw = dict(HP, master_weights=True, max_grad_norm=0.1)
    z, o = Zero1(a, AdamW8bit, **kw), AdamW8bit(b, **kw)
    for step in range(2):
        _grads(a, step)
        _grads(b, step)
        z.step()
        o.step()
    full = z.full_state_dict()
    z2 = Zero1(_params([5000, 30], torch.bfloat16), AdamW8bit, **kw)
    z2.load_full_state_dict(full)
    for p, q, r in zip(a, b, z2.params):
        assert torch.equal(p.detach(), q.detach())
        for k in ("m_q", "v_s", "exp_avg", "master"):
            if k in o.state[q]:
                assert torch.equal(z2.optimizer.state[r][k], o.state[q][k]), k


def test_capture_with_host_scalars_is_refused():
    params = _params([300], torch.float32)
    opt = AdamW(params, **HP)
    _grads(params, 1)
    opt.step()
    before = params[0].detach().clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
    assert opt.state[params[0]]["step"] == 1
    opt.step()
    assert opt.state[params[0]]["step"] == 2 and not torch.equal(before, params[0].detach())


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_capturable_steps_give_the_same_bits(cls):
    """Scalars formed on the device, with the learning rate as a number and as a tensor, through the C++ and the
    Python path."""
    made = []
    for kw in (dict(), dict(capturable=True), dict(capturable=True, lr=torch.tensor(HP["lr"], device="cuda")),
               dict(capturable=True)):
        params = _params([5000, 30, 2049], torch.bfloat16)
        made.append((params, cls(params, **dict(HP, max_grad_norm=0.1, **kw))))
    for step in range(5):
        for k, (params, o) in enumerate(made):
            _grads(params, step)
            if k == 3:
                o._slow_step(o._ready(), None)
            else:
                o.step()
    (pa, a), rest = made[0], made[1:]
    for pb, b in rest:
        for p, q in zip(pa, pb):
            assert torch.equal(p.detach(), q.detach())
            assert float(b.state[q]["step"]) == a.state[p]["step"] == 5
            for k, t in a.state[p].items():
                assert not torch.is_tensor(t) or torch.equal(t, b.state[q][k]), k
    # either kind loads the other's state
    c = cls(pa, **HP)
    c.load_state_dict(rest[0][1].state_dict())
    assert c.state[pa[0]]["step"] == 5 and type(c.state[pa[0]]["step"]) is int
    d = cls(pa, capturable=True, **HP)
    d.load_state_dict(a.state_dict())
    assert float(d.state[pa[0]]["step"]) == 5.0 and d.state[pa[0]]["step"].is_cuda


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_captured_step_replays(cls):
    """A captured step, replayed with new gradients and a new learning rate, against eager steps; eager steps in
    between and a second graph of the same optimizer."""
    lr = torch.tensor(HP["lr"], device="cuda")
    sizes = [5000, 30, 2049]
    params, plain = _params(sizes, torch.float32), _params(sizes, torch.float32)
    kw = dict(HP, max_grad_norm=0.1)
    opt, ref = cls(params, capturable=True, **dict(kw, lr=lr)), cls(plain, **kw)
    _grads(params, 0)
    _grads(plain, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    ref.step()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            opt.step()
    for step in range(1, 7):
        r = _rng(step)
        for p, q in zip(params, plain):
            q.grad = torch.from_numpy(r.normal(0, 1e-2, tuple(p.shape)).astype(np.float32)).cuda()
            p.grad.copy_(q.grad)
        value = HP["lr"] / step
        lr.fill_(value)
        ref.param_groups[0]["lr"] = float(lr)  # the fp32 number that the device reads
        if step == 4:
            opt.step()
        else:
            graphs[step % 2].replay()
        ref.step()
        assert torch.equal(opt.last_grad_norm, ref.last_grad_norm), step
        for p, q in zip(params, plain):
            assert torch.equal(p.detach(), q.detach()), step
            assert float(opt.state[p]["step"]) == ref.state[q]["step"] == step + 1
            for k, t in ref.state[q].items():
                assert not torch.is_tensor(t) or torch.equal(t, opt.state[p][k]), (k, step)


def test_captured_behind_copies_and_joined_streams():
    """What comes before the calls in a graph may be a copy, a fill, or work joined from another stream."""
    params, plain = _params([70000, 300], torch.bfloat16), _params([70000, 300], torch.bfloat16)
    kw = dict(HP, master_weights=True)
    opt, ref = AdamW8bit(params, capturable=True, **kw), AdamW8bit(plain, **kw)
    _grads(params, 0)
    _grads(plain, 0)
    opt.step()
    ref.step()
    fresh = [torch.zeros_like(p) for p in params]
    out = [tuple(torch.zeros(p.shape, device="cuda") for _ in range(2)) for p in params]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            params[1].grad.copy_(fresh[1])  # a copy on another stream
        params[0].grad.zero_()  # a fill
        main.wait_stream(side)
        grad_norm(params)
        params[0].grad.copy_(fresh[0])
        clip_grad_norm_(params, 0.5)
        opt.step()
        opt.moments(params, out=out)
    for step in range(1, 6):
        _grads(plain, step, scale=0.1)
        for f, q in zip(fresh, plain):
            f.copy_(q.grad)
        graph.replay()
        clip_grad_norm_(plain, 0.5)
        ref.step()
        want = ref.moments(plain)
        for p, q, a, b in zip(params, plain, out, want):
            assert torch.equal(p.grad, q.grad) and torch.equal(p.detach(), q.detach()), step
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), step


def test_first_step_in_a_capture_is_refused():
    params = _params([300], torch.float32)
    opt = AdamW(params, capturable=True, **HP)
    _grads(params, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="first step"):
            opt.step()
    assert not opt.state[params[0]]
    opt.step()
    half = _params([300], torch.bfloat16)
    opt2 = AdamW(half, capturable=True, **HP)
    _grads(half, 1)
    opt2.step()
    opt2.master_weights = True
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="first step"):
            opt2._plan = None
            opt2.step()
    assert "master" not in opt2.state[half[0]]
    with pytest.raises(TypeError, match="lr"):
        opt.param_groups[0]["lr"] = torch.tensor(1e-3, dtype=torch.float64, device="cuda")
        opt.step()


@pytest.mark.parametrize("block", [None, 64])
def test_master_copies_beside_fp32_parameters(block):
    """fp32 and half-precision parameters in one optimizer with master copies, a scalar and odd sizes among them."""
    shapes = [(), (3, 700), (1,), (4099,), (17, 5, 3)]
    r = _rng(12)
    params = [torch.nn.Parameter(torch.from_numpy(np.asarray(r.normal(0, 0.1, s), np.float32)).cuda().to(t))
              for t in TYPES for s in shapes]
    kw = dict(HP, master_weights=True)
    opt = AdamW(params, **kw) if block is None else AdamW8bit(params, block_size=block, min_8bit_numel=0, **kw)
    refs = [Plain32(_np(p), block) for p in params]
    for step in range(3):
        _grads(params, 40 + step)
        opt.step()
        for p, ref in zip(params, refs):
            ref.step(_np(p.grad), *ARGS)
    for p, ref in zip(params, refs):
        st = opt.state[p]
        assert ("master" in st) == (p.dtype != torch.float32)
        _check_param(_np(st.get("master", p)), ref, (p.dtype, p.shape))
        assert torch.equal(p.detach(), st.get("master", p).to(p.dtype).detach())
        if block:
            _check_codes(st, ref, (p.dtype, p.shape))


def test_refused_types_and_gradients():
    p = torch.nn.Parameter(torch.zeros(8, dtype=torch.float64, device="cuda"))
    p.grad = torch.zeros_like(p)
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        AdamW([p]).step()
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        grad_norm([p])
    q = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    q.grad = torch.zeros_like(q)
    c = torch.nn.Parameter(torch.zeros(8))
    c.grad = torch.zeros(8)
    for params in ([q, c], [c, q]):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            AdamW8bit(params).step()
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            clip_grad_norm_(params, 1.0)


@pytest.mark.parametrize("slow", [False, True])
def test_autograd_sees_the_step(slow):
    """A graph that saved a parameter cannot be run backward over its new values; nor one that saved a clipped
    gradient."""
    params = _params([300], torch.float32)
    opt = AdamW(params, **HP)
    _grads(params, 1)
    opt.step()
    loss = (params[0] * params[0]).sum()
    if slow:
        opt._slow_step(opt._ready(), None)
    else:
        opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    before = params[0].grad._version
    grad_norm(params)
    assert params[0].grad._version == before
    clip_grad_norm_(params, 1.0)
    assert params[0].grad._version > before


def test_grad_scaler_and_closure():
    params, plain = _params([3000, 7], torch.float32), _params([3000, 7], torch.float32)
    opt, ref = AdamW8bit(params, min_8bit_numel=0, **HP), AdamW8bit(plain, min_8bit_numel=0, **HP)
    scaler = torch.amp.GradScaler("cuda", init_scale=8.0)
    _grads(plain, 1)
    for p, q in zip(params, plain):
        p.grad = q.grad * 8.0
    scaler.scale(torch.zeros((), device="cuda"))
    scaler.step(opt)
    scaler.update()
    ref.step()
    assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(params, plain))
    params[0].grad = torch.full_like(params[0], float("inf"))
    before = params[1].detach().clone()
    scaler.step(opt)  # skipped
    assert torch.equal(params[1].detach(), before) and opt.state[params[0]]["step"] == 1

    def closure():
        opt.zero_grad()
        loss = sum((p * p).sum() for p in params)
        loss.backward()
        return loss

    loss = opt.step(closure)
    assert loss.requires_grad and opt.state[params[0]]["step"] == 2
    opt.zero_grad()
    opt.step()
    assert opt.state[params[0]]["step"] == 2


def test_launches_are_counted():
    params = _params([300, 5000], torch.float32)
    opt = AdamW(params, **HP)
    _grads(params, 1)
    opt.step()
    lib = _lib.load()
    before = lib.smo_launch_count()
    opt.step()
    assert lib.smo_launch_count() == before + 1  # every tensor in one launch
