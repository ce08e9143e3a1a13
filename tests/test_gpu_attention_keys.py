"""clef_paged_attention key by key: q that is not whole rows is refused."""
import pytest
import torch

import aiis_clef_b200 as clef
from test_gpu_attention import Problem

pytestmark = pytest.mark.gpu


def test_queries_that_are_not_whole_rows_are_refused(cuda_dev):
    """A remainder would come back as it was in memory."""
    p = Problem([(1, 100)], (6, 2), 128, 16, behind=0)
    at = [t.cuda() for t in (p.q, p.k, p.v, p.table, p.q_start, p.kv_len)]
    with pytest.raises(clef.ClefError, match="whole rows of 4 x 128"):
        cuda_dev.paged_attention_dev(*at, 4, 2, 128, 16, 0.1)
    with pytest.raises(clef.ClefError, match="whole rows of 6 x 256"):
        cuda_dev.paged_attention_dev(*at, 6, 2, 256, 16, 0.1)
    p.check(cuda_dev.paged_attention_dev(*at, 6, 2, 128, 16, p.scale))
