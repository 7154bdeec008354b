"""Rules of the kernels' sources that no run on a GPU may try out (CPU)."""
from __future__ import annotations

import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "drinkme_b200", "csrc")


def sources():
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            yield name, re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name,text", [s for s in sources() if "pdl_wait()" in s[1] and s[0] != "dm_device.cuh"])
def test_kernels_that_start_early_read_through_the_coherent_path(name, text):
    """A kernel that starts while its predecessor still writes (programmatic dependent launch)
    may not use loads that ask for memory nobody writes while it runs."""
    assert "__ldg(" not in text and not re.search(r"ld\.global(\.\w+)*\.nc", text), name


def test_tensor_memory_is_freed_after_the_last_product_whatever_gave_up():
    """The prompt kernel frees its tensor memory behind a wait for every product that it
    has issued, which no earlier wait's outcome skips."""
    text = dict(sources())["kv4_prompt.cu"]
    last = text[: text.index("tcgen05.dealloc")]
    at = last.rindex("mma_commit(drain, lead);")
    assert re.search(r"\n\s*mbar_wait\(drain, 0, err, kKvErrWait\);", last[at:])
    assert "if (ok)" not in last[at:]
