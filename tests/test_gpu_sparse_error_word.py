"""The error word: no bit is lost between reading and clearing it."""

import threading
import time

import pytest
import torch

from sparse_cases import i32
from tpu_cake_amd import sparse

pytestmark = pytest.mark.gpu


def test_bits_set_while_another_thread_clears(cuda):
    """One thread reads and clears all the time, another sets a bit a turn: each has to be returned by a read."""
    sparse.read_error_word(clear=True)
    seen, reads, done = 0, 0, False
    lock = threading.Lock()

    def clear():
        nonlocal seen, reads
        with torch.cuda.stream(torch.cuda.Stream()):
            while not done:
                word = sparse.read_error_word(clear=True)
                with lock:
                    seen, reads = seen | word, reads + 1

    pool = torch.zeros((2, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    x, slots = torch.ones((1, 1, 64), dtype=torch.bfloat16, device="cuda"), i32([99])
    torch.cuda.synchronize()
    thread = threading.Thread(target=clear)
    thread.start()
    lost = 0
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(400):
                with lock:
                    seen = 0
                sparse.append_kv(x, x, pool, slots)
                torch.cuda.current_stream().synchronize()
                with lock:
                    begun = reads
                deadline = time.monotonic() + 5
                while reads < begun + 2 and time.monotonic() < deadline:  # the second of them began after the bit was set
                    time.sleep(0)
                assert reads >= begun + 2
                with lock:
                    lost += seen != sparse._sparse_lib.ERR_SLOT
    finally:
        done = True
        thread.join()
    assert lost == 0
    assert sparse.read_error_word() == 0


def test_a_read_alone_clears_nothing(cuda):
    sparse.read_error_word(clear=True)
    pool = torch.zeros((2, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    x = torch.ones((1, 1, 64), dtype=torch.bfloat16, device="cuda")
    sparse.append_kv(x, x, pool, i32([99]))
    assert sparse.read_error_word() == sparse.read_error_word() == sparse._sparse_lib.ERR_SLOT
    assert sparse.read_error_word(clear=True) == sparse._sparse_lib.ERR_SLOT and sparse.read_error_word() == 0
