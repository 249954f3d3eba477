"""Kernels launched in a chain read what their parameters point to behind their wait for the kernel before them: that one may still be writing it.  No GPU: the
sources are read."""
import re

from test_chained_launches import kernels


def test_no_kernel_of_the_chain_reads_an_array_of_its_parameters_before_its_wait():
    found, ordinary = kernels()
    early = []
    for name, body in found:
        if name in ordinary:
            continue
        body = re.sub(r"\{[^{}]*\breturn;[^{}]*\}", "", body)            # ways out that wait for themselves
        waits = [body.find(wait) for wait in ("chain_wait();", "chain_begin();") if wait in body]
        before = body[:min(waits)]
        # (load_l2: values that no kernel within the last launch wrote; set-up of tensor maps takes addresses alone)
        if re.search(r"\bp\.\w+\s*\[|[=(,]\s*\*\s*\(?p\.", re.sub(r"load_l2\([^)]*\)", "", before)):
            early.append(name)
    assert not early
