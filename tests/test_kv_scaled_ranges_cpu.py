"""The block-scaled FP8 cache without a GPU, at the ends of what its calls allow."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "atlas_b200" / "csrc"


def _kernels(text):
    for m in re.finditer(r"__global__[^;{]*\{", text):
        end = text.find("\n}\n", m.end())
        yield text[m.start():m.end()].split("(")[-2].split()[-1], text[m.end():end]


@pytest.mark.parametrize("name", ["attention_scaled_tc.cu", "kv_scaled.cu", "moe.cu"])
def test_a_cluster_meets_before_it_reaches_into_shared_memory(name):
    """Another CTA's shared memory is there only once that CTA has started, which a barrier of the cluster says."""
    seen = 0
    for _, body in _kernels((CSRC / name).read_text()):
        far = re.search(r"cluster_map_shared|ld_cluster|st_cluster", body)
        if far:
            seen += 1
            assert "cluster_sync_all();" in body[:far.start()]
    assert seen
