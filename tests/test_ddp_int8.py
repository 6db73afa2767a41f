"""A model that holds 8-bit layers under DDP: rank 0's integer buffers win at the wrap and before
every training forward, together with the scales and biases that belong to them."""
import os
import socket
import traceback

import pytest
import torch
import torch.multiprocessing as mp
import torch.nn as nn


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _model(seed):
    """A trunk of two 8-bit layers (rows of no alignment in one of them), then what is trained."""
    from mxddp.models.layers import BatchNorm2d, Int8Linear, Linear

    class Net(nn.Module):
        def __init__(self):
            super().__init__()
            torch.manual_seed(seed)
            self.t1 = Int8Linear.from_linear(Linear(20, 33, fuse_relu=True))
            self.t2 = Int8Linear.from_linear(Linear(33, 16, bias=False))
            self.bn = BatchNorm2d(4)
            self.head = Linear(16, 5)
            self.register_buffer("kinds", torch.tensor([[seed, 2], [3, 4]], dtype=torch.int32))
            self.register_buffer("flags", torch.tensor([seed > 1, True, False]))
            self.register_buffer("empty", torch.zeros(0, 3, dtype=torch.int64))
            self.register_buffer("elsewhere", torch.zeros(3, dtype=torch.int32, device="meta"), persistent=False)
            self.register_buffer("count_elsewhere", torch.zeros((), dtype=torch.int64, device="meta"), persistent=False)
            self.bn.num_batches_tracked.fill_(seed)

        def trunk(self, x):
            return self.t2(self.t1(x))

        def forward(self, x):
            h = self.trunk(x).reshape(-1, 4, 2, 2)
            return self.head(self.bn(h).reshape(-1, 16))

    return Net()


def _worker(rank, ws, port, gpu, broadcast, q):
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(ws),
                          LOCAL_RANK=str(rank), LOCAL_WORLD_SIZE=str(ws))
        from mxddp.parallel import comm
        from mxddp.parallel.ddp import DistributedDataParallel as DDP

        if gpu:
            comm.init_distributed(use_gpu=True)
        else:
            comm.init_distributed(rank=rank, world_size=ws, use_gpu=False, init_method=f"tcp://127.0.0.1:{port}")
        dev = torch.device("cuda", 0) if gpu else torch.device("cpu")
        x = torch.randn(6, 20, generator=torch.Generator().manual_seed(3)).to(dev)
        model = _model(1 + rank)
        meta = {n: b for n, b in model.named_buffers() if b.is_meta}
        for n in meta:
            delattr(model, n)
        model.to(dev)
        for n, b in meta.items():
            model.register_buffer(n, b, persistent=False)
        ddp = DDP(model, broadcast_buffers=broadcast)
        out = []

        def keep():
            with torch.no_grad():
                y = model.trunk(x)
            out.append(({k: v.cpu().clone() for k, v in model.state_dict().items()}, y.cpu()))

        keep()  # after the wrap
        if rank == 0:  # rank 0 alone takes other weights
            model.load_state_dict({k: v for k, v in _model(7).state_dict().items() if not k.startswith("head")},
                                  strict=False)
        ddp(x).sum().backward()
        keep()
        ddp.eval()
        if rank == 0:
            with torch.no_grad():
                model.t1.weight.neg_()
        ddp(x)
        keep()  # no broadcast without training
        q.put((rank, None, [({k: v.numpy() for k, v in sd.items()}, y.numpy()) for sd, y in out]))
        if gpu:
            torch.cuda.synchronize()
        comm.shutdown()
    except Exception:
        q.put((rank, traceback.format_exc(), None))


def _run(gpu, broadcast):
    ws = 2
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    ps = [ctx.Process(target=_worker, args=(r, ws, port, gpu, broadcast, q)) for r in range(ws)]
    for p in ps:
        p.start()
    out = {}
    try:
        for _ in range(ws):
            r, err, res = q.get(timeout=100)
            assert err is None, f"rank {r}: {err}"
            out[r] = [({k: torch.from_numpy(v) for k, v in sd.items()}, torch.from_numpy(y)) for sd, y in res]
    finally:
        for p in ps:
            p.join(timeout=30)
            if p.is_alive():
                p.kill()
    return out[0], out[1]


@pytest.mark.parametrize("gpu", [pytest.param(False, id="gloo"), pytest.param(True, marks=pytest.mark.gpu, id="peer")])
def test_rank_0_has_the_integer_buffers(gpu):
    a, b = _run(gpu, True)
    want = [_model(1), _model(7)]
    for i in (0, 1):
        (sa, ya), (sb, yb) = a[i], b[i]
        w = want[i].state_dict()
        for k in sa:
            if k.startswith("t") or k in ("kinds", "flags"):
                assert torch.equal(sa[k], w[k]) and torch.equal(sb[k], w[k]), (i, k)
        assert torch.equal(ya, yb)
    # the counter: rank 0's at the wrap, each rank's own steps from there
    assert [int(s["bn.num_batches_tracked"]) for s in (a[0][0], b[0][0], a[1][0], b[1][0])] == [1, 1, 8, 2]
    assert torch.equal(a[2][0]["t1.weight"], -want[1].t1.weight) and torch.equal(b[2][0]["t1.weight"], want[1].t1.weight)


def test_no_buffers_broadcast():
    a, b = _run(False, False)
    assert torch.equal(a[0][0]["t1.weight"], _model(1).t1.weight)
    assert torch.equal(b[0][0]["t1.weight"], _model(2).t1.weight)
    assert int(b[0][0]["bn.num_batches_tracked"]) == 2
