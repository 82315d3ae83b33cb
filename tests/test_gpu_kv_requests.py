"""GPU checks that a request on the cache's pages is served as a whole or not at
all."""
import pytest

from test_gpu_kv_pages import Model, i32, make, pages  # noqa: F401  (pages: the fixture)
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,bad", [(4, [0, 9]), (4, [1, -1, 0]), (2000, list(range(0, 1999, 2)) + [2000])])
def test_free_with_one_index_out_of_range_frees_nothing(pages, seqs, bad):  # noqa: F811
    t, m = make(pages, 3 * seqs, seqs, 3, layers=1), Model(3 * seqs, seqs, 3, 16)
    who, more = list(range(seqs)), [1 + 7 * s % 40 for s in range(seqs)]
    t.extend(i32(who), i32(more), sum(more))
    m.extend(who, more)
    t.free(i32(bad))
    m.compare(t)
    with pytest.raises(RuntimeError, match="index"):
        t.check()
    good = [s for s in bad if 0 <= s < seqs]
    t.free(i32(good + good[:1]))
    m.free(good)
    m.compare(t)
    t.check()


def test_free_in_a_graph(pages):  # noqa: F811
    t, m = make(pages, 64, 8, 4, layers=1), Model(64, 8, 4, 16)
    who = i32([1, 3, 3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.free(who)
    for names in ([1, 3, 3], [2, 8, 0], [0, 0, 2]):
        t.extend(i32([0, 1, 2, 3]), i32([20, 5, 16, 33]), 74)
        m.extend([0, 1, 2, 3], [20, 5, 16, 33])
        who.copy_(i32(names))
        graph.replay()
        if max(names) < 8:
            m.free(names)
            t.check()
        else:
            with pytest.raises(RuntimeError, match="index"):
                t.check()
        m.compare(t)
        t.free(i32([0, 1, 2, 3]))
        m.free([0, 1, 2, 3])


@pytest.mark.parametrize("more,total", [([3], 5), ([3], 2), ([-1], 0)])
def test_the_message_names_a_wrong_total(pages, more, total):  # noqa: F811
    t, m = make(pages, 8, 4, 3, layers=1), Model(8, 4, 3, 16)
    assert t.extend(i32([2]), i32(more), total).tolist() == [-1] * total
    with pytest.raises(RuntimeError, match="add up"):
        t.check()
    m.compare(t)
