"""The data-parallel step of a model with a norm on both sides of its blocks, on CPU: two gloo ranks against one process that holds both ranks'
batches.  The junction gives the gradients of layer l's second norm and gate and of layer l + 1's first norm at once, which lie in two buckets."""
import os
import socket
import sys

import pytest
import torch
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _cfg(gate):
    from train_gpt_b200.step import SMALL, StepConfig
    return StepConfig(**SMALL, mm="bf16", norm="torch_reference", loss="torch", optimizer="torch", activation="relu2", block_norm="sandwich", residual_gate=gate,
                      residual_scale=0.9)


def _worker(rank, world, port, gate, out_dir):
    sys.path.insert(0, ROOT)
    import torch.distributed as dist
    from train_gpt_b200.step import Trainer, synthetic_batch
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.manual_seed(0)
    cfg = _cfg(gate)
    tr = Trainer(cfg, "cpu", world_size=world, seed=0)
    ids, tgt = synthetic_batch(cfg, 2, "cpu", seed=100 + rank, learnable=True)
    done, exchanged, before = [], [], []
    launch, exchange = tr.buckets._launch, tr.buckets._exchange
    tr.buckets._launch = lambda bi: (done.append(bi), launch(bi))[1]
    tr.buckets._exchange = lambda bi: (exchanged.append(bi), before.append(list(done)), exchange(bi))[2]
    loss, norm = tr.step(ids, tgt)
    torch.save({"loss": loss, "norm": norm, "grads": [f.clone() for f in tr.buckets.flat], "params": [p.detach().clone() for p in tr.model.parameters()],
                "done": done, "exchanged": exchanged, "before": before}, os.path.join(out_dir, f"rank{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_two_ranks_match_one_with_both_batches(gate, tmp_path):
    from train_gpt_b200.step import Trainer, synthetic_batch
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.start_processes(_worker, args=(2, port, gate, str(tmp_path)), nprocs=2, join=True, start_method="spawn")
    a, b = (torch.load(tmp_path / f"rank{r}.pt") for r in range(2))
    cfg = _cfg(gate)
    # every bucket complete once, from the head to the embeddings, and exchanged once after that
    assert a["done"] == b["done"] == list(range(2 + cfg.n_layers)) == a["exchanged"] == b["exchanged"]
    assert all(bi in seen for bi, seen in zip(a["exchanged"], a["before"]))
    for name in ("grads", "params"):
        assert all(torch.equal(p, q) for p, q in zip(a[name], b[name]))
    assert torch.equal(a["norm"], b["norm"])

    tr = Trainer(cfg, "cpu", world_size=1, seed=0)
    batches = [synthetic_batch(cfg, 2, "cpu", seed=100 + r, learnable=True) for r in range(2)]
    tr.buckets.zero()
    loss = tr.model.loss(*(torch.cat(t) for t in zip(*batches)))
    loss.backward()
    tr.buckets.finish()
    # the mean of two means over equal batches: float32 losses below 8, their logits of 2^-8 in bf16, the same ones in both
    assert abs(float(loss.detach()) - 0.5 * (float(a["loss"]) + float(b["loss"]))) <= 2.0 ** -10
    scale = min(1.0, cfg.clip_norm / (float(a["norm"]) + 1e-6))                # the ranks' gradients are kept after the clip
    for bi, (full, dp) in enumerate(zip(tr.buckets.flat, a["grads"])):
        # parameter by parameter: gradients are bf16 sums, over the batch in one and added from two halves and scaled in the other: three roundings
        # of 2^-8 apart, beside those of the sums inside (whose order the batch changes), as many again
        for want, got in zip(tr.buckets.views(bi, full), tr.buckets.views(bi, dp)):
            want = want.float() * scale
            assert float((got.float() - want).norm()) <= 6 * 2.0 ** -8 * float(want.norm()) and float(want.norm()) > 0
