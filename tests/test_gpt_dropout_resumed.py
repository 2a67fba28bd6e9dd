"""A decoder with dropout goes on from a checkpoint with the masks that the uninterrupted job draws; every rank draws its own."""
import os
import socket

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from parameter_server_b200.models.gpt import GPT, GPTConfig

CPU = dict(n_layer=1, d_model=32, n_head=4, d_ff=40, vocab=64, seq_len=16, fused=True, gated=True, rotary=True)
GPU = dict(n_layer=2, d_model=256, n_head=4, d_ff=680, vocab=512, seq_len=64, lr=3e-3, weight_decay=0.0, fused=True, gated=True, rotary=True)


def test_a_checkpoint_has_the_masks_place(tmp_path):
    model = GPT(GPTConfig(**CPU, dropout=0.1), device="cpu", seed=3)
    model.drop_passes = 41
    model.save_checkpoint(str(tmp_path / "a"))
    other = GPT(GPTConfig(**CPU, dropout=0.1), device="cpu", seed=9)
    assert other.drop_seed != model.drop_seed
    other.load_checkpoint(str(tmp_path / "a") + "/")
    assert (other.drop_seed, other.drop_passes) == (model.drop_seed, 41)
    # saved again with another count, and by a model that drops nothing
    model.drop_passes = 42
    model.save_checkpoint(str(tmp_path / "a"))
    other.load_checkpoint(str(tmp_path / "a"))
    assert other.drop_passes == 42
    plain = GPT(GPTConfig(**CPU), device="cpu", seed=5)
    plain.save_checkpoint(str(tmp_path / "a"))
    other.load_checkpoint(str(tmp_path / "a"))
    assert (other.drop_seed, other.drop_passes) == (plain.drop_seed, 0)


def test_a_checkpoint_without_the_masks_place_leaves_it_alone(tmp_path):
    """As they were written before checkpoints had it."""
    model = GPT(GPTConfig(**CPU, dropout=0.1), device="cpu", seed=3)
    model.save_checkpoint(str(tmp_path))
    for name in os.listdir(tmp_path):
        if not name.startswith("table_"):
            os.remove(tmp_path / name)
    other = GPT(GPTConfig(**CPU, dropout=0.1), device="cpu", seed=9)
    other.drop_passes, seed = 7, other.drop_seed
    other.load_checkpoint(str(tmp_path))
    assert (other.drop_seed, other.drop_passes) == (seed, 7)


@pytest.mark.parametrize("seed", [-1, 1 << 47, (1 << 63) - 1])
def test_seeds_of_any_size(tmp_path, seed):
    model = GPT(GPTConfig(**CPU, dropout=0.1), device="cpu", seed=seed)
    model.save_checkpoint(str(tmp_path))
    other = GPT(GPTConfig(**CPU, dropout=0.1), device="cpu")
    other.load_checkpoint(str(tmp_path))
    assert other.drop_seed == model.drop_seed == (seed << 16) & 0xFFFFFFFFFFFFFFFF


def test_a_count_of_another_whole_number_type(tmp_path):
    model, other = (GPT(GPTConfig(**CPU, dropout=0.1), device="cpu") for _ in range(2))
    model.drop_passes, model.drop_seed = np.int64(41), torch.tensor(5)
    model.save_checkpoint(str(tmp_path))
    other.load_checkpoint(str(tmp_path))
    assert (other.drop_seed, other.drop_passes) == (5, 41)


def _rank(rank, world, port, uri):
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    model = GPT(GPTConfig(**CPU, dropout=0.1), device="cpu", seed=3)
    model.drop_passes = 5
    seeds = [None] * world
    dist.all_gather_object(seeds, model.drop_seed)
    assert len(set(seeds)) == world
    model.save_checkpoint(uri)
    other = GPT(GPTConfig(**CPU, dropout=0.1), device="cpu", seed=8)
    other.load_checkpoint(uri)
    assert (other.drop_seed, other.drop_passes) == (seeds[rank], 5)
    dist.barrier()
    dist.destroy_process_group()


def test_every_rank_has_masks_of_its_own(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_rank, (2, port, str(tmp_path)), nprocs=2)


@pytest.mark.gpu
def test_a_job_goes_on_as_if_nothing_had_happened(tmp_path):
    data = torch.randint(0, 512, (8, 65), generator=torch.Generator().manual_seed(0)).cuda()
    tokens, targets = data[:, :-1], data[:, 1:]
    model = GPT(GPTConfig(**GPU, dropout=0.2), seed=1)
    for _ in range(2):
        model.train_step(tokens, targets)
    model.save_checkpoint(str(tmp_path))
    other = GPT(GPTConfig(**GPU, dropout=0.2), seed=2)
    other.load_checkpoint(str(tmp_path))
    losses = [[m.forward(tokens, targets)[1].item() for _ in range(2)] for m in (model, other)]
    assert losses[0] == losses[1] and losses[0][0] != losses[0][1]
    other.check()
