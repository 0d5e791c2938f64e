"""The 8-bit cache in the engine and around it: status words, models, generated tokens."""
from types import SimpleNamespace as NS

import pytest
import torch

gpu = pytest.mark.gpu


def test_the_step_reads_the_status_word_of_its_own_device(monkeypatch):
    """A process whose first kernels ran on another device: waits that give up in this device's attention are reported, too."""
    from vllm_kunlun_b200.engine.runner import ModelRunner
    from vllm_kunlun_b200.ops import _ext
    words = {0: NS(device=torch.device("cuda:0")), 1: NS(device=torch.device("cuda:1"))}
    monkeypatch.setattr(_ext, "available", lambda: True)
    monkeypatch.setattr(_ext, "C", lambda: NS(gemm_status_tensor=lambda device=None: words.get(0 if device is None else device)))

    def read(device):
        runner = NS(pstate=NS(tp_comm=None), device=torch.device(device), _status_cache=None)
        return [w for _, w in ModelRunner._status_words(runner)]
    assert read("cuda:0") == [words[0]]
    assert read("cuda:1") == [words[0], words[1]]
    assert read("cuda:2") == [words[0]]            # nothing of the kind has run there


@gpu
def test_status_words_by_device():
    from test_kv8 import attend, batch
    from vllm_kunlun_b200.ops import _ext, gemm_cuda
    attend(batch([1], [40], 4, 2, 128, 64, torch.bfloat16, "cuda"))
    word = _ext.C().gemm_status_tensor()
    here = _ext.C().gemm_status_tensor(torch.cuda.current_device())
    assert here is not None and here.device.index == torch.cuda.current_device()
    assert _ext.C().gemm_status_tensor(torch.cuda.device_count()) is None
    assert word is not None and int(here) == 0
    here.fill_(905)
    try:
        with pytest.raises(RuntimeError):
            gemm_cuda.check_status()
    finally:
        here.zero_()
    gemm_cuda.check_status()
