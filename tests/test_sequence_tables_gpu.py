"""The embedding's gradient over tables of many rows: where a token and its index no longer fit one 32-bit number, and
where the sort takes one to four digits."""
import pytest
import torch

from . import blocks_plain as P
from . import sequence_plain as Q
from .test_sequence_gpu import rand, whole

pytestmark = pytest.mark.gpu

AT = 524287  # rows from which on a key of 13 bits less takes more than 32


def tokens_of(V, N, seed):
    """Spread over the table, at both of its ends, the same one many times, and some outside."""
    t = whole(0, V, N, seed=seed)
    t[::7], t[1::11], t[2::13], t[3::17] = V - 1, 0, V // 2, V
    t[4::19] = whole(max(0, V - 5), V, t[4::19].numel(), seed=seed + 1)
    t[5::23] = -1
    return t


def check(ms, N, V, D, into, seed=1):
    """Named rows against their sums in 64 bits; all others are zero, or what they were."""
    t, dout = tokens_of(V, N, seed), rand(N, D, seed=seed + 5)
    table = rand(V, D, seed=seed + 6) if into else torch.zeros(V, D, device="cuda")
    on = (t >= 0) & (t < V)
    rows, at = t[on].unique(return_inverse=True)
    add, slack = Q.embedding_gradient(dout[on].double(), at, rows.numel(), 0.5)
    want = table[rows].double() + add
    if into:  # the sum is added to what is there: one rounding of the result more
        slack = slack + Q.EPS32 * (want.abs() + slack)
    A = ms.from_torch
    if into:
        held = table.clone()
        ms.embedding_backward(A(dout), A(t), scale=0.5, into=A(held))
    else:
        held = ms.embedding_backward(A(dout), A(t), rows=V, scale=0.5).torch()
    P.close(held[rows], want, slack, "named rows")
    held[rows], table[rows] = 0.0, 0.0
    assert torch.equal(held, table)


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("N", [129, 4097, 8192])
@pytest.mark.parametrize("V", [AT - 1, AT, AT + 1, 600000])
def test_keys_of_more_than_32_bits(ms, V, N, into):
    check(ms, N, V, 4, into)


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("V", [1, 511, 512, (1 << 18) - 1, 1 << 18, 1 << 27])
def test_digits(ms, V, into):
    """Tokens outside are one more key: from 512 rows on that takes two digits of up to nine bits, from 2^18 three, from 2^27 four."""
    check(ms, 9001, V, 1 if V > 1 << 20 else 5, into)


def test_rows_that_share_their_low_digits(ms):
    """Tokens that differ in their highest digit alone, and repeat in one order."""
    V, N = 1 << 20, 10000
    t = torch.arange(N, device="cuda") % 8 * (V // 8) + 3
    dout = rand(N, 4, seed=1)
    got = ms.embedding_backward(ms.from_torch(dout), ms.from_torch(t), rows=V).torch()
    want, slack = Q.embedding_gradient(dout.double(), t, V, 1.0)
    P.close(got, want, slack)


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("N", [128 * 2048, 128 * 2048 + 1, 1_500_001])
def test_many_tokens(ms, N, into):
    """Around the number of tiles from which their counts are scanned, and far above."""
    check(ms, N, 32000, 2, into)


def test_time_grows_with_the_tokens(ms):
    """Four times the tokens take four times as long; where every block reads the counts of all it is sixteen (7.5 with the
    rest of the call). Least times of some runs, six times allowed."""
    def least(N):
        t, dout = ms.from_torch(whole(0, 32000, N, seed=1)), ms.from_torch(torch.zeros(N, 8, device="cuda", dtype=torch.bfloat16))
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ms.embedding_backward(dout, t, rows=32000)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert least(1 << 24) < 6 * least(1 << 22)
