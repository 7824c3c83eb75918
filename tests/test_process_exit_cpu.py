"""How a rank of the command line ends: its process group goes before the interpreter does (CPU, gloo)."""
import os
import subprocess
import sys

import pytest
import torch
import torch.distributed as dist

from multimodal_seq2seq_gscan_amd import __main__ as command

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RANK = """
import sys, torch
import torch.distributed as dist
from multimodal_seq2seq_gscan_amd.__main__ import _end_distributed
sys.setswitchinterval(5.0)             # a transport thread that wants the interpreter lock does not get it in passing
rank, path = int(sys.argv[1]), sys.argv[2]
dist.init_process_group("gloo", store=dist.FileStore(path, 2), rank=rank, world_size=2)
for _ in range(200):
    dist.all_reduce(torch.ones(1000))
_end_distributed()
_end_distributed()                     # nothing left to end
assert not dist.is_initialized()
"""


def test_ranks_end_their_group_and_leave_normally(tmp_path):
    """Without the group's end about one rank in seven aborts here (-6) after its work was done."""
    for k in range(6):
        ranks = [subprocess.Popen([sys.executable, "-c", RANK, str(r), str(tmp_path / f"store{k}")], cwd=ROOT, text=True,
                                  stdout=subprocess.PIPE, stderr=subprocess.STDOUT) for r in range(2)]
        logs = [p.communicate(timeout=120)[0] for p in ranks]
        assert [p.returncode for p in ranks] == [0, 0], logs


def _one_rank(path):
    dist.init_process_group("gloo", store=dist.FileStore(str(path), 1), rank=0, world_size=1)
    return 0, 1


@pytest.mark.parametrize("owned", [True, False])
def test_training_ends_the_group_that_it_created(tmp_path, monkeypatch, owned):
    """`--mode=train` ends the group that it created, and leaves one that was there before it."""
    from multimodal_seq2seq_gscan_amd import train
    calls = []
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(train, "train_on_dataset", lambda **flags: calls.append(dist.is_initialized()))
    store = tmp_path / "store"
    if owned:
        monkeypatch.setattr(command, "_init_distributed", lambda: _one_rank(store))
    else:
        _one_rank(store)
        monkeypatch.setattr(command, "_init_distributed", lambda: (0, 1))
    try:
        flags = vars(command.build_parser().parse_args(["--mode", "train", "--output_directory", str(tmp_path / "out")]))
        command.main(flags)
        assert calls == [True]
        assert dist.is_initialized() is (not owned)
    finally:
        if dist.is_initialized():
            dist.destroy_process_group()
