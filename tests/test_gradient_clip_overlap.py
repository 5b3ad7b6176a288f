"""Results of clipping that share memory, without a GPU: tensors whose elements do not fill their memory are compared element by element with the plain definition,
a mark on every byte."""
import itertools

import pytest
import torch

from basedxl_amd import gradient_clip


def marked(t):
    """The bytes of a buffer that a view of it holds, each as often as it is held."""
    offsets = [t.storage_offset() * t.element_size()]
    for n, st in zip(t.shape, t.stride()):
        offsets = [o + i * st * t.element_size() for o in offsets for i in range(n)]
    return [o + i for o in offsets for i in range(t.element_size())]


BUFFER = torch.zeros(4096, dtype=torch.uint8)
WORDS, HALVES = BUFFER.view(torch.float32), BUFFER.view(torch.bfloat16)
VIEWS = {
    "left": WORDS.view(32, 32)[:, :3], "right": WORDS.view(32, 32)[:, 3:7], "across": WORDS.view(32, 32)[:, 2:5], "all": WORDS.view(32, 32), "turned": WORDS.view(32, 32).t(),
    "even": WORDS[::2], "odd": WORDS[1::2], "thirds": WORDS[1::3], "row": WORDS.view(32, 32)[5], "low_halves": HALVES[::2], "high_halves": HALVES[1::2],
    "halves_of_even": HALVES.view(-1, 4)[:, :2], "middle": HALVES.view(-1, 4)[:, 1:3], "blocks": WORDS.view(8, 4, 32)[::2, 1:3, ::5], "other_blocks": WORDS.view(8, 4, 32)[1::2, 1:3, ::5],
    "one": WORDS[77:78], "last": WORDS[1023:], "empty": WORDS[5:5], "rows": WORDS.as_strided((6, 9), (64, 2), 3), "slanted": WORDS.as_strided((6, 9), (65, 2), 4), "knight": WORDS.as_strided((2, 2), (3, 2), 11),
    "windows": WORDS.as_strided((6, 3), (1, 1), 40), "spread": WORDS.as_strided((5, 4), (0, 1), 9), "folded": WORDS.as_strided((4, 4, 2), (3, 9, 18), 0), "wide": WORDS.as_strided((3, 4, 2), (1, 3, 12), 200),
}


@pytest.mark.parametrize("name", VIEWS)
def test_elements_of_one_tensor(name):
    bytes_ = marked(VIEWS[name])
    assert gradient_clip._overlaps_itself(VIEWS[name]) == (len(set(bytes_)) < len(bytes_))


@pytest.mark.parametrize("first, second", itertools.combinations_with_replacement(VIEWS, 2))
def test_elements_of_two_tensors(first, second):
    want = bool(set(marked(VIEWS[first])) & set(marked(VIEWS[second])))
    assert gradient_clip._overlap(VIEWS[first], VIEWS[second]) == want == gradient_clip._overlap(VIEWS[second], VIEWS[first])


def refused(gradients, results):
    try:
        gradient_clip._refuse_shared_memory(gradients, results)
    except ValueError as e:
        assert "share" in str(e) and "memory" in str(e)
        return True
    return False


def test_lists():
    v, far = VIEWS, torch.zeros(32, 32)
    other = lambda t: torch.zeros_like(t, memory_format=torch.contiguous_format)   # noqa: E731
    assert not refused([v["left"], v["right"]], [v["left"], v["right"]])                                # side by side, in place
    assert refused([v["left"], v["across"]], [v["left"], v["across"]])                                  # a column of both, at other addresses
    assert refused([far[:, 1:4].clone(), far], [v["across"], v["all"]])                                 # a result in another
    assert refused([v["left"], other(v["left"])], [other(v["left"]), v["left"]])                        # a result in another's gradient
    assert refused([other(v["across"]), v["row"]], [v["across"], other(v["row"])])                      # ... in part
    assert not refused([v["left"], v["across"]], [other(v["left"]), other(v["across"])])                # gradients may share
    assert not refused([v["all"]], [v["turned"]]) and not refused([v["left"]], [v["left"]])             # a result in its own gradient
    assert refused([v["even"], v["low_halves"][1:]], [v["even"], other(v["low_halves"][1:])])           # half a word of another type's
    assert refused([other(v["windows"])], [v["windows"]]) and refused([other(v["spread"])], [v["spread"]])
    assert not refused([v["empty"], v["empty"]], [v["empty"], v["empty"]])


def test_many_columns():
    """Columns of a buffer, all of whose ranges lie over each other."""
    wide = torch.zeros(100000, 60)
    columns = [wide[:, i:i + 1] for i in range(60)]
    assert not refused(columns, columns) and refused(columns, columns[:-1] + [wide[:, 0:1]])
