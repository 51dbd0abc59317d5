"""Views of one buffer whose byte ranges cross: `share_no_byte` against the sets of bytes that they hold."""
import random

import torch

from intent_amd.runtime.torch_views import byte_span, share_no_byte
from intent_amd.runtime.invocation import ViewFacts


def facts(view):
    begin, end = byte_span(view.data_ptr(), tuple(view.shape), tuple(view.stride()), view.element_size())
    return ViewFacts(tuple(view.shape), tuple(view.stride()), view.data_ptr(), None, None, None, view.dtype, begin, end, None)


def held(view):
    places = torch.tensor(0)
    for n, stride in zip(view.shape, view.stride()):
        places = (places[..., None] + torch.arange(n) * stride)
    at = view.data_ptr() + view.element_size() * places.flatten()
    return set((at[:, None] + torch.arange(view.element_size())).flatten().tolist())


def test_never_wrong():
    """Random strided views of a small buffer, of elements of one to four bytes: what is called apart is apart."""
    rng, buffer, apart, crossing = random.Random(1), torch.zeros(4096, dtype=torch.uint8), 0, 0
    types = (torch.uint8, torch.float16, torch.float32)
    for _ in range(4000):
        steps = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 32]) for _ in range(3)]
        pair = []
        for _ in range(2):
            dtype = rng.choice(types)
            strides = [s if rng.random() < 0.8 else rng.randint(0, 40) for s in steps]
            pair.append(buffer.view(dtype).as_strided([rng.randint(1, 5) for _ in range(3)], strides, rng.randint(0, 40)))
        left, right = (facts(v) for v in pair)
        if not (left.begin < right.end and right.begin < left.end):
            continue
        crossing += 1
        said = share_no_byte(left, right)
        assert said == share_no_byte(right, left)
        apart += said
        assert not said or not held(pair[0]) & held(pair[1])
    assert crossing > 2000 and apart > 100


def test_packed_buffers():
    packed = torch.zeros((9, 40, 64), dtype=torch.float16)
    assert share_no_byte(facts(packed[:, :32]), facts(packed[:, 32:]))
    assert not share_no_byte(facts(packed[:, :33]), facts(packed[:, 32:]))
    pages = torch.zeros((5, 2, 16, 3, 64), dtype=torch.uint8)
    assert share_no_byte(facts(pages[:, 0]), facts(pages[:, 1]))
    assert share_no_byte(facts(pages[:, 0].transpose(1, 2)), facts(pages[:, 1]))
    assert not share_no_byte(facts(pages[:, 0]), facts(pages[:, 0]))
    assert not share_no_byte(facts(pages[:4]), facts(pages[1:]))
    beside = torch.zeros((5, 16, 3, 2, 64), dtype=torch.uint8)
    assert share_no_byte(facts(beside[..., 0, :]), facts(beside[..., 1, :]))
    assert not share_no_byte(facts(beside[..., 0, :]), facts(beside[..., 0, 63:]))
    columns = torch.zeros((6, 8))
    assert share_no_byte(facts(columns[:, ::2]), facts(columns[:, 1::2]))
    assert not share_no_byte(facts(columns[:, 1:]), facts(columns[:, :-1]))
    assert not share_no_byte(facts(columns[:1].expand(6, 8)), facts(columns))
