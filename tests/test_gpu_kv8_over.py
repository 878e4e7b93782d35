"""A captured append of the 8-bit cache replayed after its batch is over: it stores nothing, and rounds nothing that
the begun blocks hold."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import filled, plain, rows_of

pytestmark = pytest.mark.gpu


def captured(nh, lens, stream=None):
    """(cache, ids, graph, its k and v): one row for each sequence, in the middle of a block, captured and replayed once."""
    rng = np.random.default_rng(sum(lens))
    c, ids, _, _ = filled(nh, rng, lens, 2, 64, 64, 64, "f32", layers=2, extra_pages=6)
    k, v = (rows_of(rng, len(lens), 2, 64, "f32").cuda() for _ in range(2))
    c.extend(ids, [1] * len(lens))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for layer in (0, 1):
            c.append(layer, k, v)
    graph.replay()
    torch.cuda.synchronize()
    return c, ids, graph, k, v


def held(c, ids):
    return [plain(x) for x in c.read(None, ids, [0] * len(ids), [c.length(s) for s in ids])]


@pytest.mark.parametrize("form", ["truncate", "truncate another", "fork", "free"])
def test_a_replay_after_the_batch(nh, form):
    c, ids, graph, k, v = captured(nh, [70, 5, 40])
    if form == "truncate":
        c.truncate(ids[0], 70)
    elif form == "truncate another":
        c.truncate(ids[2], 3)
    elif form == "fork":
        ids += c.fork(ids[0], 2)
    else:
        c.free(ids[1])
        ids[1] = c.new_seq()
    was = held(c, ids)
    k.fill_(50.0)
    v.fill_(-50.0)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held(c, ids), was):
            assert np.array_equal(x, y)
    # the next batch of that shape is the graph's again
    some = ids[:3]
    c.extend(some, [1, 1, 1])
    graph.replay()
    torch.cuda.synchronize()
    n = [c.length(s) for s in some]
    now = c.read(1, some, [x - 1 for x in n], [1, 1, 1])
    # (a step is less than twice the row's own 50 / 127)
    assert bool(((now[0] - 50.0).abs() <= 50 / 127).all()) and bool(((now[1] + 50.0).abs() <= 50 / 127).all())


def test_on_another_stream(nh):
    c, ids, graph, k, v = captured(nh, [70, 5])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.truncate(ids[0], 70, stream=side)
    with torch.cuda.stream(side):
        k.fill_(50.0)
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    x = held(c, ids)
    assert np.abs(x[0]).max() < 49.0


def test_changes_in_a_capture_are_refused_and_change_nothing(nh):
    c, ids, graph, k, v = captured(nh, [70, 5])
    was, lens, room = held(c, ids), [c.length(s) for s in ids], c.free_pages
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        for call in (lambda: c.truncate(ids[0], 3), lambda: c.fork(ids[0]), lambda: c.free(ids[1])):
            with pytest.raises(nh.NeedleHipError):
                call()
        k.fill_(2.0)
    assert [c.length(s) for s in ids] == lens and c.free_pages == room and c.rows == 2
    for x, y in zip(held(c, ids), was):
        assert np.array_equal(x, y)
    # refused for another reason: the batch lives on
    for call in (lambda: c.truncate(ids[0], 100), lambda: c.free(7), lambda: c.fork(ids[0], 1000)):
        with pytest.raises(nh.NeedleHipError):
            call()
    k.fill_(25.0)
    graph.replay()
    torch.cuda.synchronize()
    assert bool(((c.read(0, ids[:1], [70], [1])[0] - 25.0).abs() <= 25 / 127).all())
