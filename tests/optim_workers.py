"""Importable worker for the spawned multi-process AdamW tests."""

import os

import torch

from dist_workers import _small_cfg
from util_dist import init_env


def adamw_twice_worker(rank, world, port, outdir, mode, model, norm, bits):
    """The same short run twice: parameters and events of each."""
    init_env(rank, world, port)
    from eventgrad_amd.config import TriggerConfig
    from eventgrad_amd.train.trainer import Trainer

    runs = []
    for cycle in range(2):
        os.environ["MASTER_PORT"] = str(port + 1 + cycle)
        cfg = _small_cfg(mode, model=model, epochs=1, lr=2e-3,
                         dataset="synthetic-mnist" if model == "cnn2"
                         else "synthetic",
                         n_train=64 if model == "cnn2" else 16,
                         batch_size=8 if model == "cnn2" else 4,
                         trigger=TriggerConfig(adaptive=True, horizon=1.05,
                                               initial_comm_passes=2))
        cfg.norm = norm
        cfg.optim.optimizer = "adamw"
        cfg.optim.state_bits = bits
        cfg.optim.weight_decay = 0.01
        tr = Trainer(cfg)
        assert tr.space.momentum is None
        m = tr.train()
        runs.append((tr.space.param.clone(), m.num_events_total,
                     tr.engine.opt.steps))
        torch.distributed.destroy_process_group()
    torch.save({"runs": runs}, os.path.join(outdir, f"adamw_r{rank}.pt"))
