"""Keys and values in 8 bits at their edges: scratch, queries and scales of unusual sizes, masks that part two query tiles, bytes that nobody sees."""

import subprocess
import sys

import pytest
import torch

from nkipy_b200 import ops
from nkipy_b200.ops import _lib
from nkipy_b200.ops import quantized_kv as Q
from tests.test_quantized_kv import pool, shuffled_table


# ------------------------------------------------------------------------------------------------ scratch
class Library:
    """Stands in for the kernel library: sizes are right once it is initialised."""

    def __init__(self, sms=148):
        self.sms, self.ready = sms, False

    def nkb_init(self):
        self.ready = True
        return 0

    def nkb_q8_attn_decode_scratch_floats(self, *sizes):
        return 1000 if self.ready else 10

    def nkb_q8_attn_prefill_scratch_floats(self, *sizes):
        return 2000 if self.ready else 20


@pytest.fixture
def fresh_library(monkeypatch):
    """A library that no call has reached yet, and sizes that no call has asked for."""
    def forget():
        Q._decode_floats.cache_clear()
        Q._prefill_floats.cache_clear()

    fake = Library()
    forget()
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    monkeypatch.setattr(_lib, "_initialised", False)
    yield fake
    forget()


def test_sizes_of_scratch_are_asked_of_an_initialised_library(fresh_library):
    assert Q._decode_floats(1, 8, 128, 4, 4) == 1000
    fresh_library.ready = _lib._initialised = False
    assert Q._prefill_floats(1, 100, 32, 8, 128, 32) == 2000


def test_no_size_is_kept_of_a_library_without_a_device(fresh_library, monkeypatch):
    monkeypatch.setattr(fresh_library, "nkb_init", lambda: -1)
    for _ in range(2):
        with pytest.raises(_lib.KernelLibraryError):
            Q._decode_floats(1, 8, 128, 4, 4)
        with pytest.raises(_lib.KernelLibraryError):
            Q._prefill_floats(1, 100, 32, 8, 128, 32)


@pytest.mark.gpu
def test_scratch_of_a_new_process():
    """A cache that is the process's first use of the library has room for what its steps take."""
    code = """
from nkipy_b200 import ops
from nkipy_b200.ops import _lib, quantized_kv as Q
sizes = [(8, 32, 1, 32), (8, 32, 1, 250), (1, 16, 3, 400), (4, 4, 2, 77)]
first = [Q.decode_scratch(ops.QuantizedPages.new(1, nkv, 128, "cuda"), nq, batch, pages).numel() for nkv, nq, batch, pages in sizes]
_lib.ensure_init()
Q._decode_floats.cache_clear()
again = [Q.decode_scratch(ops.QuantizedPages.new(1, nkv, 128, "cuda"), nq, batch, pages).numel() for nkv, nq, batch, pages in sizes]
assert first == again, (first, again)
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


@pytest.mark.gpu
def test_kernels_refuse_scratch_that_is_too_small(monkeypatch):
    """The library looks at the size by itself: here the caller believes in a smaller one."""
    g = torch.Generator().manual_seed(1)
    table, blocks = shuffled_table(g, [900])
    k, v = pool(g, blocks, 2, 64, "cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")       # noqa: E731
    q = torch.zeros((1, 4 * 64), dtype=torch.bfloat16, device="cuda")
    small = torch.zeros((Q.COUNTERS + 8,), device="cuda")
    monkeypatch.setattr(Q, "_decode_floats", lambda *sizes: small.numel())
    with pytest.raises(_lib.KernelLibraryError):
        ops.paged_attn_decode(q, k, v, table.cuda(), i32(900), 0.1, num_splits=4, scratch=small)
    monkeypatch.setattr(Q, "_prefill_floats", lambda *sizes: small.numel())
    monkeypatch.setattr(Q, "_scratch", lambda *a: small)
    with pytest.raises(_lib.KernelLibraryError):
        ops.flash_attn_prefill(q, k, v, table.cuda(), i32(0), i32(1), i32(900), 0.1, max_q_len=1)
    assert not bool(small.any())
