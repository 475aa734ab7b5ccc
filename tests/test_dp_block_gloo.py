"""The data-parallel step of a model with rotary positions, normed queries and keys and a gated feed-forward, on CPU: two gloo ranks against one
process that holds both ranks' batches; and with dropout, whose masks differ from rank to rank."""
import os
import socket
import sys

import pytest
import torch
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _cfg(dropout):
    from train_gpt_b200.step import SMALL, StepConfig
    return StepConfig(**SMALL, mm="bf16", norm="torch_reference", loss="torch", optimizer="torch", activation="swiglu", positions="rotary", qk_norm=True, dropout=dropout)


def _worker(rank, world, port, dropout, out_dir):
    sys.path.insert(0, ROOT)
    import torch.distributed as dist
    from train_gpt_b200.step import Trainer, synthetic_batch
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.manual_seed(0)
    cfg = _cfg(dropout)
    tr = Trainer(cfg, "cpu", world_size=world, seed=0)
    ids, tgt = synthetic_batch(cfg, 2, "cpu", seed=100 + (rank if dropout == 0 else 0), learnable=True)
    loss, norm = tr.step(ids, tgt)
    torch.save({"loss": loss, "norm": norm, "grads": [f.clone() for f in tr.buckets.flat], "params": [p.detach().clone() for p in tr.model.parameters()],
                "seed": None if tr.model.dropout_seed is None else int(tr.model.dropout_seed)}, os.path.join(out_dir, f"rank{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


def _run(dropout, tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.start_processes(_worker, args=(2, port, dropout, str(tmp_path)), nprocs=2, join=True, start_method="spawn")
    return [torch.load(tmp_path / f"rank{r}.pt") for r in range(2)]


def test_two_ranks_match_one_with_both_batches(tmp_path):
    from train_gpt_b200.step import Trainer, synthetic_batch
    a, b = _run(0.0, tmp_path)
    for name in ("grads", "params"):
        assert all(torch.equal(p, q) for p, q in zip(a[name], b[name]))
    cfg = _cfg(0.0)
    tr = Trainer(cfg, "cpu", world_size=1, seed=0)
    batches = [synthetic_batch(cfg, 2, "cpu", seed=100 + r, learnable=True) for r in range(2)]
    tr.buckets.zero()
    loss = tr.model.loss(*(torch.cat(t) for t in zip(*batches)))
    loss.backward()
    tr.buckets.finish()
    assert abs(float(loss.detach()) - 0.5 * (float(a["loss"]) + float(b["loss"]))) <= 2.0 ** -10
    scale = min(1.0, cfg.clip_norm / (float(a["norm"]) + 1e-6))
    for bi, (full, dp) in enumerate(zip(tr.buckets.flat, a["grads"])):
        # bf16 sums, over the batch in one and added from two halves and scaled in the other: three roundings of 2^-8 apart, and as many for the sums inside
        for want, got in zip(tr.buckets.views(bi, full), tr.buckets.views(bi, dp)):
            want = want.float() * scale
            assert float((got.float() - want).norm()) <= 6 * 2.0 ** -8 * float(want.norm()) and float(want.norm()) > 0


def test_every_rank_draws_masks_of_its_own(tmp_path):
    """The same batch on both ranks: the losses differ, the exchanged gradients and the parameters do not."""
    a, b = _run(0.5, tmp_path)
    assert b["seed"] - a["seed"] == 1 << 40 and float(a["loss"]) != float(b["loss"])
    for name in ("grads", "params"):
        assert all(torch.equal(p, q) for p, q in zip(a[name], b[name]))
