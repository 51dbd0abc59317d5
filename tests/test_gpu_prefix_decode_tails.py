"""paged_gqa_decode_prefix where a run of tokens ends inside a step of 32: an infinite value of its last token gives an infinity, whatever the
keys behind it read. Only places that the infinity reaches may change, so the rest is compared bit for bit with the run without it."""
import pytest
import torch

from tests.gpu_util import announce
from tests.test_gpu_prefix_decode import case, i32, kernel, run

pytestmark = pytest.mark.gpu

# prefix, own lengths, query heads, key heads, d, page: runs of whole and of partial steps, pages of whole tiles of 32, of 16, and others; one
# and two tiles of query rows a wave.
CASES = [(1, [1, 3], 4, 2, 64, 16), (31, [31, 33], 8, 2, 128, 32), (33, [32, 7], 8, 1, 64, 7), (64, [64, 65], 4, 2, 128, 16), (3, [1, 31], 6, 2, 64, 64),
         (100, [45, 160], 8, 2, 128, 24), (1000, [300, 1], 4, 2, 64, 1), (129, [20, 17] * 20, 16, 2, 64, 16), (97, [33, 5] * 10, 32, 4, 128, 20),
         (161, [1, 70] * 20, 8, 1, 128, 32)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("prefix,lengths,heads,kv_heads,d,ps", CASES)
def test_infinite_last_value(device, dtype, prefix, lengths, heads, kv_heads, d, ps):
    announce("decode behind a prefix, infinite last value", dtype, prefix, len(lengths), heads, kv_heads, d, ps)
    given = case(prefix + d, dtype, prefix, lengths, heads, kv_heads, d, ps, size=0.5)
    want = run(device, dtype, given)
    assert want.isfinite().all()
    group = heads // kv_heads
    last_of_prefix = (int(given[3][(prefix - 1) // ps]), (prefix - 1) % ps)
    own = len(lengths) - 1
    last_of_own = (int(given[6][int(given[5][own]) + (lengths[own] - 1) // ps]), (lengths[own] - 1) % ps)
    for at, sequences in ((last_of_prefix, slice(None)), (last_of_own, slice(own, None))):
        for sign in (1.0, -1.0):
            values = given[2].clone()
            values[at[0], at[1], 0, :3] = sign * float("inf")
            got = run(device, dtype, [*given[:2], values, *given[3:]])
            assert (got[sequences, :group, :3] == sign * float("inf")).all()
            keep = torch.ones(got.shape, dtype=torch.bool, device=device)
            keep[sequences, :group, :3] = False
            assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_no_score_is_a_number_above_minus_infinity(device, dtype):
    """A row all of whose scores are -inf has no attention: exp(-inf + inf) is not a number. Where only the prefix or only its own tokens are
    so, the others count alone."""
    announce("decode behind a prefix, all scores -inf", dtype)
    given = list(case(8, dtype, 45, [40, 3, 0], 8, 2, 128, 16))
    given[0][:, :4] = given[0][:, :4].abs() + 0.5
    shared, own = given[3].long(), given[6].long()
    everywhere, in_prefix, in_own = (given[1].clone() for _ in range(3))
    everywhere[:, :, 0] = float("-inf")
    in_prefix[shared, :, 0] = float("-inf")
    in_own[own, :, 0] = float("-inf")
    want = run(device, dtype, given)
    got = run(device, dtype, [given[0], everywhere, *given[2:]])
    assert got[:, :4].isnan().all() and torch.equal(got[:, 4:], want[:, 4:])
    got = run(device, dtype, [given[0], in_prefix, *given[2:]])
    alone = run(device, dtype, [*given[:4], torch.zeros_like(given[4]), *given[5:]])
    assert torch.equal(got[:2, :4], alone[:2, :4]) and got[2, :4].isnan().all()
    got = run(device, dtype, [given[0], in_own, *given[2:]])
    alone = run(device, dtype, [*given[:7], torch.zeros_like(given[7]), given[8]])
    assert torch.equal(got[:, :4], alone[:, :4])


@pytest.mark.parametrize("ps", [4095, 4096])
def test_as_many_tokens_as_a_length_counts(device, ps):
    """2^31 - 1 own tokens, whose pages are one: equal keys and values of powers of two, so the output is those values exactly, whatever
    the order of the sums."""
    announce("decode behind a prefix, 2^31 - 1 tokens", ps)
    length, d = 2 ** 31 - 1, 64
    positions = -(-length // ps)
    q = torch.ones((1, 1, d), dtype=torch.bfloat16, device=device)
    keys = torch.zeros((1, ps, 1, d), dtype=torch.bfloat16, device=device)
    values = (2.0 ** (torch.arange(d, device=device) % 7 - 3)).bfloat16().expand(1, ps, 1, d).contiguous()
    tables = [i32(v).to(device) for v in ([], [0], [0, positions])]
    pages = torch.zeros(positions, dtype=torch.int32, device=device)
    got = kernel("bf16", 1).run(q, keys, values, *tables, pages, i32([length]).to(device), 0.125)
    assert torch.equal(got[0, 0], values[0, 0, 0])
