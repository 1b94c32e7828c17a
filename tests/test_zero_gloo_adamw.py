"""ZeRO-1 with AdamW and AdamW8bit on CPU ranks (gloo, world_size 2): partition, refusals, and states gathered to one
rank and loaded at another world size.  The CUDA step cannot run on the CPU: the states are made by hand."""

import os
import socket
from datetime import timedelta

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from smo_optimizer_b200 import AdamW, AdamW8bit, zero

SHAPES = [(64, 256), (128, 128), (32, 32), (300,), (256, 64), (96, 96), (10,)]
KW = {AdamW: dict(lr=0.5, master_weights=True), AdamW8bit: dict(lr=0.5, master_weights=True, block_size=64)}


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _params(dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(0)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype)) for s in SHAPES]


def _state(i, p, cls):
    """The state of tensor i, with values that tell it from any other."""
    g = torch.Generator().manual_seed(100 + i)
    st = {"step": 7 + i, "master": torch.randn(p.shape, generator=g)}
    if cls is AdamW8bit and p.numel() >= 4096:
        nb = -(-p.numel() // 64)
        st.update(m_q=torch.randint(-127, 128, (nb, 64), generator=g).to(torch.int8), m_s=torch.rand(nb, 1, generator=g),
                  v_q=torch.randint(0, 256, (nb, 64), generator=g).to(torch.uint8), v_s=torch.rand(nb, 1, generator=g))
    else:
        st.update(exp_avg=torch.randn(p.shape, generator=g), exp_avg_sq=torch.rand(p.shape, generator=g))
    return st


def _same(a, b):
    assert a.keys() == b.keys()
    for k, t in a.items():
        assert (t.dtype == b[k].dtype and torch.equal(t, b[k])) if torch.is_tensor(t) else t == b[k], k


def _run(rank, cls, reduce_grads):
    """Owners of the tensors and, on rank 0, the gathered state."""
    params = _params()
    with pytest.raises(ValueError, match="max_grad_norm"):
        zero.Zero1(params, cls, max_grad_norm=1.0, reduce_grads=reduce_grads, **KW[cls])
    z = zero.Zero1(params, cls, reduce_grads=reduce_grads, **KW[cls])
    for i, p in enumerate(params):
        if z.owner[i] == rank:
            z.optimizer.state[p] = _state(i, p, cls)
    full = z.full_state_dict()
    assert (full is None) == (rank != 0)
    box = [full]
    dist.broadcast_object_list(box, src=0)
    fresh = _params()
    z2 = zero.Zero1(fresh, cls, **KW[cls])
    z2.load_full_state_dict(box[0])
    for i, p in enumerate(fresh):
        if z2.owner[i] == rank:
            _same(z2.optimizer.state[p], _state(i, p, cls))
        else:
            assert z2.optimizer is None or p not in z2.optimizer.state
    return list(z.owner), full


COMBINATIONS = [(cls, reduce_grads) for cls in (AdamW, AdamW8bit) for reduce_grads in (False, True)]


def _worker(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=20))
    try:
        out[rank] = ("ok", [_run(rank, *c) for c in COMBINATIONS])
    except BaseException as e:  # reported to the parent
        out[rank] = ("error", repr(e))
    finally:
        dist.destroy_process_group()


def test_two_ranks():
    ctx = mp.get_context("spawn")
    out = ctx.Manager().dict()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, out)) for r in range(2)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=120)
        if p.is_alive():
            p.kill()
            pytest.fail("a rank did not finish")
    assert out[0][0] == out[1][0] == "ok", (out[0], out[1])
    for (cls, _), (owner, full), (other, _) in zip(COMBINATIONS, out[0][1], out[1][1]):
        assert owner == other and set(owner) == {0, 1}
        # the costs that the partition goes by
        costs = [zero.adamw_step_bytes(s, cls is AdamW8bit, KW[cls].get("block_size", 128), elem=2, master=True)
                 for s in SHAPES]
        assert owner == zero.lpt_partition(costs, 2)
        # one process loads what two gathered
        params = _params()
        opt = cls(params, **KW[cls])
        opt.load_state_dict(full)
        for i, p in enumerate(params):
            _same(opt.state[p], _state(i, p, cls))
