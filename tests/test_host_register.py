"""cbm_host_register: what it refuses, and that a caller learns whether a buffer was page-locked."""
import ctypes as C
import mmap
import os
import sys

import numpy as np
import pytest

import cleanba_amd.lib as L

HERE = os.path.dirname(os.path.abspath(__file__))
PAGE = mmap.PAGESIZE


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.SO_PATH):
        L.build()
    return L.load()


@pytest.fixture
def hole():
    """The address of three pages whose middle one is not mapped."""
    libc = C.CDLL(None)
    libc.mmap.restype, libc.mmap.argtypes = C.c_void_p, [C.c_void_p, C.c_size_t, C.c_int, C.c_int, C.c_int, C.c_long]
    libc.munmap.argtypes = [C.c_void_p, C.c_size_t]
    at = libc.mmap(None, 3 * PAGE, mmap.PROT_READ | mmap.PROT_WRITE, mmap.MAP_PRIVATE | mmap.MAP_ANONYMOUS, -1, 0)
    libc.munmap(at + PAGE, PAGE)
    yield at
    libc.munmap(at, PAGE)
    libc.munmap(at + 2 * PAGE, PAGE)


def refused(lib, h, ptr, n, text):
    assert lib.cbm_host_register(h, C.c_void_p(ptr), C.c_int64(n)) == -1
    assert text in lib.cbm_last_error().decode()


def test_refuses_what_is_no_buffer(lib, hole):
    refused(lib, None, 0, 100, "empty buffer")
    refused(lib, None, hole, 0, "empty buffer")
    refused(lib, None, hole, -5, "empty buffer")
    refused(lib, None, hole + PAGE, 10, "not mapped")
    refused(lib, None, hole + 10, PAGE, "not mapped")            # runs into the hole
    refused(lib, None, hole + 2 * PAGE - 1, 100, "not mapped")   # begins in it
    refused(lib, None, hole, 2 ** 63 - 1, "not mapped")
    refused(lib, None, hole, PAGE, "null context")
    big = np.zeros(5000 * PAGE + 7, np.uint8)                    # (more pages than are asked about at once)
    refused(lib, None, big.ctypes.data, big.nbytes, "null context")


def test_trainer_takes_a_refused_buffer_for_pageable(monkeypatch, tmp_path):
    """A buffer that could not be page-locked is tried once and not un-registered; one whose registration raises likewise."""
    sys.path.insert(0, HERE)
    from oracle_engine import OracleEngine
    from cleanba_amd import trainer
    from cleanba_amd.args import parse_args
    calls, gone = [], []

    def engine(answer):
        class Eng(OracleEngine):
            def host_register(self, arr):
                calls.append(arr.ctypes.data)
                if answer is None:
                    raise L.CbmError("refused")
                return answer

            def host_unregister(self, arr):
                gone.append(arr.ctypes.data)
        return Eng

    monkeypatch.chdir(tmp_path)
    argv = ["--local-num-envs", "4", "--num-actor-threads", "1", "--num-steps", "4", "--env-backend", "host", "--network", "nature",
            "--total-timesteps", "32", "--log-frequency", "1000", "--update-epochs", "1", "--num-minibatches", "2"]
    for answer in (True, False, None):
        del calls[:], gone[:]
        trainer.train(parse_args(argv, "ppo"), "ppo", engine_factory=engine(answer))
        assert calls and len(calls) == len(set(calls))
        assert sorted(gone) == (sorted(calls) if answer else [])


@pytest.mark.gpu
def test_a_caller_learns_what_became_of_the_buffer(lib, hole):
    import torch
    cfg = L.default_config(L.ALGO_PPO)
    cfg.local_num_envs, cfg.num_actor_slots, cfg.num_steps, cfg.num_minibatches, cfg.update_epochs = 1, 1, 8, 1, 1
    ctx = L.Context(cfg)
    try:
        refused(lib, ctx.h, hole, 3 * PAGE, "not mapped")
        arr = np.zeros(1 << 20, np.uint8)
        for _ in range(2):
            locked = ctx.host_register(arr)
            assert locked in (True, False)
            x = torch.arange(1000, device="cuda")                # no error is left for the next call
            assert int(x.sum()) == 499500
            ctx.sync()
            ctx.host_unregister(arr)
    finally:
        ctx.close()
