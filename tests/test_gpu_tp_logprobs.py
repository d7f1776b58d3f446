"""nf_tp_logprobs on a row-split linear over one, two and all GPUs: every rank reads the whole gathered output, whichever of
the two gather buffers holds it.  Tolerances as in test_gpu_stack_verify.py's test of one rank: the logits' F32 sums of K
terms, twice, and the log-probabilities' own 1e-5."""
import datetime
import os
import socket
import sys

import numpy as np
import pytest

from helpers import REPO, nfm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
SHAPES = [(1000, 256, 3), (40003, 64, 2), (7, 64, 1), (4099, 512, 9)]  # (rows of the linear, columns, tokens)
TOP = 5


def make_case(i):
    rows, cols, tokens = SHAPES[i]
    g = torch.Generator().manual_seed(200 + i)
    return (torch.randn(rows, cols, generator=g).bfloat16(), torch.randn(tokens, cols, generator=g),
            torch.randint(0, rows, (tokens,), generator=g).int())


def rank_main(rank, world, port, out_dir, transport):
    sys.path.insert(0, str(REPO / "tests"))
    os.environ["NF_TP_TRANSPORT"] = transport
    import torch
    import torch.distributed as dist

    torch.cuda.set_device(rank)
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world,
                            timeout=datetime.timedelta(seconds=60))
    mm = nfm()
    gid = [mm.ep_group_id() if rank == 0 and world > 1 else None]
    dist.broadcast_object_list(gid, src=0)
    tp = mm.TpGroup(max_tokens=9, max_rows=40003, rank=rank, world=world, group_id=gid[0], device=rank)
    res, s = {}, torch.cuda.Stream()
    for i, (rows, cols, tokens) in enumerate(SHAPES):
        w, x, target = make_case(i)
        r0, r1 = tp.split(rows)
        w, x, target = w[r0:r1].contiguous().cuda(), x.cuda(), target.cuda()
        lp, en, tl = (torch.empty(n, device="cuda") for n in ((tokens,), (tokens,), (tokens, TOP)))
        ti = torch.empty(tokens, TOP, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        tp.linear_bf16(w, rows, cols, x, tokens, stream=s.cuda_stream)
        tp.logprobs(tokens, rows, target, lp, en, ti, tl, stream=s.cuda_stream)
        tp.sync(s.cuda_stream)
        for name, t in (("lp", lp), ("en", en), ("ti", ti), ("tl", tl)):
            res[f"{name}{i}"] = t.cpu().numpy()
    np.savez(os.path.join(out_dir, f"r{rank}.npz"), **res)
    dist.barrier()  # every rank's last call is done before any handle of the group goes
    tp.close()
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("ranks, transport", [("one", "nvlink"), ("two", "nvlink"), ("two", "nccl"), ("all", "nvlink")])
def test_logprobs_of_a_split_linear(tmp_path, ranks, transport):
    n = torch.cuda.device_count()
    world = {"one": 1, "two": 2, "all": min(n, 8)}[ranks]
    if n < 2 and ranks != "one":
        pytest.skip("needs 2 GPUs")
    if ranks == "all" and world == 2:
        pytest.skip("only two GPUs: covered by the two-rank case")
    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.start_processes(rank_main, args=(world, port, str(tmp_path), transport), nprocs=world, start_method="spawn", join=True)
    for r in range(world):
        got = np.load(tmp_path / f"r{r}.npz")
        for i, (rows, cols, tokens) in enumerate(SHAPES):
            w, x, target = (t.double() if t.is_floating_point() else t.long() for t in make_case(i))
            full = torch.log_softmax(x @ w.T, -1)
            tol = 2 * cols * 2.0 ** -24 * float((x.abs() @ w.abs().T).max()) + 1e-5
            top = full.topk(TOP)
            assert np.array_equal(got[f"ti{i}"], top.indices.numpy()), (r, i)
            assert np.abs(got[f"lp{i}"] - full.gather(1, target[:, None])[:, 0].numpy()).max() <= tol
            assert np.abs(got[f"tl{i}"] - top.values.numpy()).max() <= tol
            assert np.abs(got[f"en{i}"] + (full.exp() * full).sum(-1).numpy()).max() <= 10 * tol
