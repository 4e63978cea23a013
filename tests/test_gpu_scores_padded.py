"""Prompts whose documents do not begin with the first row or do not end with the last, against the definition in 64 bits."""
import pytest
import torch
from test_gpu_pages import generator
from test_gpu_scores import K, run  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap,alibi,window,sinks", [(None, False, None, 0), (20.0, True, None, 0), (None, True, 100, 5)])
@pytest.mark.parametrize("s,h,hkv,documents,prefix", [(1024, 4, 2, [400, 1024], 0), (1024, 1, 1, [400, 1024], 0), (2048, 4, 2, [400, 2048], 1500), (1300, 2, 1, [1200, 1210], 60), (385, 4, 4, [384, 385], 0),
                                                      (700, 2, 2, [128, 129, 700], 0), (1100, 8, 8, [700, 900], 10)])
def test_documents_that_begin_late(K, s, h, hkv, documents, prefix, softcap, alibi, window, sinks):
    """In front of them lie whole tiles of queries, which go through no keys."""
    for _ in range(3):
        got, seen = run(K, generator(s), s, h, hkv, window, sinks, 0, softcap, alibi, documents, None, prefix)
        assert not got[~seen.any(1)].any()


def test_offsets_that_do_not_rise_end(K):
    """What comes is undefined; every call ends without an error, and the next one is right."""
    from test_gpu_pages import D, normal
    r, g = torch.Generator().manual_seed(3), generator(3)
    q, k, v = normal(g, 1500, 4, D), normal(g, 1500, 2, D), normal(g, 1500, 2, D)
    for i in range(60):
        documents = torch.randint(-100, 1600, (1 + i % 7,), generator=r, dtype=torch.int32).cuda()
        K.causal_attn(q, k, v, documents=documents, prefix=[0, 1000][i % 2], window=[None, 150][i % 3 == 0], sinks=[0, 300][i % 5 == 0])
        assert K.tc_error_flag() == 0
    run(K, g, 700, 4, 2, documents=[300, 700])


@pytest.mark.parametrize("documents", [[0, 1000], [1500, 2600], [3999, 4000], [0, 0], [2049, 2050, 2300]])
def test_rows_of_none_are_zeros_in_many_blocks(K, documents):
    """Each time: what comes into a block's memory for queries that see nothing must not come out."""
    from test_gpu_pages import D, normal
    g = generator(4)
    q, k, v = normal(g, 4000, 32, D), normal(g, 4000, 8, D), normal(g, 4000, 8, D)
    where = torch.tensor(documents, dtype=torch.int32, device="cuda")
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(200):
        got = K.causal_attn(q, k, v, documents=where)
        wrong += got[:documents[0]].count_nonzero() + got[documents[-1]:].count_nonzero()
    assert wrong.item() == 0 and K.tc_error_flag() == 0
