"""Paged attention where batches and contents are unusual."""
import pytest

from test_paged_gpu import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,H,G", [
    ([(128, 2048)] * 13 + [(1, 32768)], 16, 4), ([(1, 2048)] * 63 + [(1, 4096)], 2, 2),
    ([(32, 1000)] * 60 + [(1, 40000)], 32, 8), ([(2, 700)] * 40 + [(1, 30000)], 8, 4)])
def test_equal_lengths_and_one_long_sequence(cuda, seqs, H, G):
    run(cuda, seqs, H, G, 128, page=64)
