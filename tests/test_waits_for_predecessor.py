"""The cache's kernels, which may start before the one ahead of them is done, by their source: none of a CTA's ways out is ahead of the wait for that one.  A CTA that left
without it would let the kernel behind begin while the one ahead still writes; that is nothing a run shows."""
import os

import pytest

from test_cluster_meetings import CSRC, _bodies


def _kernels() -> list:
    found = []
    for name in sorted(os.listdir(CSRC)):
        if name.endswith(".cu") and (name.startswith("attention") or name == "kv_cache.cu"):
            with open(os.path.join(CSRC, name)) as f:
                for kernel, body in _bodies(f.read()):
                    if "pdl_wait()" in body:
                        found.append(pytest.param(body, id=kernel))
    return found


def test_the_kernels_are_found():
    assert {p.id for p in _kernels()} >= {"attention_decode_kernel", "attention_chunk_kernel", "attention_f32_kernel", "join_kernel", "join_pieces_kernel",
                                          "expand_kernel", "append_kernel", "read_kernel"}


@pytest.mark.parametrize("body", _kernels())
def test_no_way_out_ahead_of_the_wait(body):
    assert "return;" not in body[:body.index("pdl_wait()")]
