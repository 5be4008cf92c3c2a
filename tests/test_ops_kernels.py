"""Every kernel over rows of logits that is built has a call that launches it: the library's symbols
against the cuts of rows that calls can have (no GPU needed)."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from luminamoon_amd.ops import backend as B

SHAPES = [(64, 4), (64, 8), (256, 8), (512, 8), (512, 13), (1024, 8), (1024, 16)]
UNITS = 256  # compute units of the card


def _cut(vector, rows, vocab, top, grad):
    """(threads, vectors, slices) of a call whose rows start on words."""
    slices = 0
    for threads, vectors in SHAPES:
        if threads == 64 and top > 48:
            continue
        if not grad and threads > 512 and (vectors > 8 or rows >= 4 * UNITS):
            break
        if vocab <= threads * vectors * vector:
            slices = 1
            break
    if slices == 0:
        for threads, vectors in reversed(SHAPES[2:] if grad else SHAPES[2:4]):
            slices = -(-vocab // (threads * vectors * vector))
            if rows * slices >= UNITS:
                break
    if not grad and (threads, vectors) == (512, 8) and (top or slices == 1) and rows * slices >= 8 * UNITS:
        threads, vectors = 256, 16
    return threads, vectors, slices


def test_no_kernel_is_built_that_no_call_reaches():
    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("nm not available")
    if not os.path.exists(B.LIB_PATH):
        from luminamoon_amd import build_ext

        build_ext.build_ops()
    text = subprocess.run([nm, "-C", B.LIB_PATH], check=True, capture_output=True, text=True).stdout
    found = re.findall(r" lvops::rows_kernel<lvops::(\w+), (\d+), (\d+), \(lvops::Way\)(\d), (\w+), (\w+)>", text)
    built = {(t, int(a), int(b), int(way), top == "true", grad == "true") for t, a, b, way, top, grad in found}
    reached = set()
    for name, vector in (("F32", 4), ("BF16", 8), ("F16", 8)):
        for rows in (1, 2, 40, 300, 1023, 1024, 3000, 100_000):
            for vocab in sorted({threads * vectors * vector + d for threads, vectors in SHAPES for d in (0, 1)} | {300_000, 10 ** 7}):
                for top in (0, 1, 48, 49, 128):
                    reached.add((name, *_cut(vector, rows, vocab, top, False)[:2], 0, top > 0, False))
                reached.add((name, *_cut(vector, rows, vocab, 0, False)[:2], 1, False, False))
                threads, vectors, slices = _cut(vector, rows, vocab, 0, True)
                reached.add((name, threads, vectors, 1, False, slices == 1))
    assert built - reached == set(), "built, but no call has such a cut"
    assert reached - built == set(), "a call without a kernel"
