"""Beam selection against a full sort in 64 bits: parents and tokens equal, scores rounded once."""
import numpy as np
import pytest
import torch
import kv4_reference as ref
from gpu_helpers import Guarded, dev, host

pytestmark = pytest.mark.gpu
LOWEST = np.finfo(np.float32).min


def check(logits, scores, beams, k, finished=None, eos=0, logits_dev=None):
    from tenzo_b200 import kernels
    want_parent, want_token, want_score = ref.select(logits, scores, beams, k, finished, eos)
    g, groups = Guarded(), len(scores) // beams
    ws = g.empty((int(kernels.load_library().tenzo_cuda_beam_select_workspace_bytes(groups, beams, logits.shape[1], k)),), torch.uint8)
    got = kernels.beam_select(dev(logits) if logits_dev is None else logits_dev, dev(scores), beams=beams, k=k, finished=None if finished is None else dev(finished),
                              eos=eos, workspace=ws)
    parent, token, score = (host(t) for t in got)
    g.check()
    assert np.array_equal(parent, want_parent) and np.array_equal(token, want_token), (parent, want_parent, token, want_token)
    both = np.isfinite(want_score)
    assert np.array_equal(both, np.isfinite(score)) and np.array_equal(score[~both], want_score[~both].astype(np.float32))
    # Rounded once to fp32 (2^-24), and the logarithm of the sum is good to 2^-19: an exponential that is taken in 32 bits counts where the logit is
    # d <= ln(vocab) < 12 below the largest (those further off have no weight), so that its exponent d log2(e), below 18, is rounded by 2^-20 or 0.7 2^-20 of the
    # exponential, log2(e) in 24 bits is off by 1.4e-8 d or 0.2 2^-20, and the hardware's 2^x by 2^-22. All that is 1.2 2^-20 if all logits went the same
    # way, and half of it is the largest's weight at d = 12; below d = 8 it is 0.8 2^-20. A thread's sum of 32 is rounded 31 times by 2^-24
    # of what has come together, half the sum on average: 1 2^-20 at most.
    assert (abs(score[both] - want_score[both]) <= 2.0 ** -24 * abs(want_score[both]) + 2.0 ** -19).all()
    return parent, token, score


@pytest.mark.parametrize("groups,beams,vocab,k", [
    (1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 5, 15), (1, 4, 1024, 8), (3, 2, 1000, 4), (2, 5, 8191, 10), (1, 3, 8192, 3), (1, 3, 8193, 6), (2, 32, 4001, 64), (1, 1, 50001, 64),
    (1, 4, 128256, 8), (5, 8, 30011, 16), (70, 2, 2048, 4), (1, 16, 333, 32), (300, 1, 77, 1), (2, 12, 50001, 24), (1, 2, 300007, 4),
])
def test_shapes(cuda_lib, groups, beams, vocab, k):
    rng = np.random.default_rng(vocab + k)
    logits = (rng.standard_normal((groups * beams, vocab)) * 2.5).astype(np.float32)
    scores = (-20 - 3 * rng.random(groups * beams)).astype(np.float32)
    check(logits, scores, beams, k)


@pytest.mark.parametrize("vocab", [64, 1023, 20000, 128256])
def test_masked_tokens(cuda_lib, vocab):
    """Masks of -infinity, of the lowest number and of NaN; rows with fewer tokens left than are asked for, with one, and with none."""
    rng = np.random.default_rng(vocab)
    beams, k = 6, 12
    logits = (rng.standard_normal((2 * beams, vocab)) * 3).astype(np.float32)
    logits[0, rng.random(vocab) < 0.9] = -np.inf
    logits[1] = -np.inf
    logits[2] = -np.inf
    logits[2, vocab - 1] = 1.5
    logits[3, rng.random(vocab) < 0.5] = np.nan
    logits[4] = LOWEST
    logits[4, [3, 5]] = -2.0
    logits[5] = np.nan
    logits[6] = LOWEST                                   # every token alike: uniform
    logits[7, 10:] = -np.inf
    logits[8] = -np.inf
    logits[8, : 5] = [1, 1, 1, 1, 1]
    scores = (-5 * rng.random(2 * beams)).astype(np.float32)
    check(logits, scores, beams, k)


def test_rows_with_nothing_left(cuda_lib):
    """All beams masked, dead (score -inf or NaN), or both: the lowest indices, at -infinity."""
    rng = np.random.default_rng(0)
    logits = rng.standard_normal((9, 500)).astype(np.float32)
    logits[:3] = -np.inf
    scores = np.array([-1, -2, -3, -np.inf, -np.inf, -np.inf, -np.inf, np.nan, -4], np.float32)
    logits[8, 3:] = -np.inf
    parent, token, score = check(logits, scores, 3, 6)
    assert (score[:2] == -np.inf).all() and (parent[:2] == 0).all() and (token[:2] == np.arange(6)).all()
    assert (score[2, 3:] == -np.inf).all()


def test_ties(cuda_lib):
    """Equal logits within a row, equal rows, zeros of both signs, first steps (all beams alike, all but one dead): the lowest index first."""
    rng = np.random.default_rng(1)
    vocab = 9001
    row = np.round(rng.standard_normal(vocab) * 2).astype(np.float32)
    same = np.tile(row, (4, 1))
    check(same, np.full(4, -1.0, np.float32), 4, 8)
    check(same, np.array([0, -np.inf, -np.inf, -np.inf], np.float32), 4, 8)
    check(np.zeros((4, vocab), np.float32), np.zeros(4, np.float32), 4, 64)
    check(np.full((4, vocab), -7.25, np.float32), np.array([-1, 0, 0, -1], np.float32), 4, 64)
    signs = np.where(rng.random((2, vocab)) < 0.5, -0.0, 0.0).astype(np.float32)
    signs[:, ::3] = -1
    check(signs, np.zeros(2, np.float32), 2, 64)


def test_many_large_values_side_by_side(cuda_lib):
    """The largest logits lie next to one another, or a fixed distance apart (whatever way the row is dealt out, some threads hold many), ascending or descending."""
    rng = np.random.default_rng(2)
    vocab = 20011
    for step in (1, 4, 32, 128, 256, 512, 1024, 2048):
        logits = rng.standard_normal((4, vocab)).astype(np.float32)
        at = (7 + step * np.arange(2000)) % vocab
        logits[:, at] += 50 + np.arange(2000, dtype=np.float32) / 64
        logits[2:] = logits[2:, ::-1]
        check(logits, np.zeros(4, np.float32), 2, 64)
    ramp = np.arange(vocab, dtype=np.float32)
    check(np.stack([ramp, -ramp, ramp[::-1], np.sin(ramp)]), np.zeros(4, np.float32), 4, 64)


def test_extreme_numbers(cuda_lib):
    rng = np.random.default_rng(3)
    logits = (rng.standard_normal((4, 3000)) * 1e4).astype(np.float32)
    logits[1] = rng.standard_normal(3000).astype(np.float32) * np.float32(1e-40)        # denormals
    logits[2, 17] = np.inf
    logits[2, 900] = np.inf
    logits[3, 5] = np.finfo(np.float32).max
    check(logits, np.array([-1e6, 0, -1e30, 3.0], np.float32), 4, 8)
    check(logits, np.zeros(4, np.float32), 1, 8)


def test_finished_beams(cuda_lib):
    rng = np.random.default_rng(4)
    beams, vocab, k = 4, 700, 8
    logits = rng.standard_normal((3 * beams, vocab)).astype(np.float32)
    scores = (-30 + 5 * rng.random(3 * beams)).astype(np.float32)
    finished = np.zeros(3 * beams, np.int32)
    finished[[0, 2, 3]] = 1
    finished[4:8] = 5                                   # all of a group: their end tokens, then the lowest indices at -infinity
    scores[2], scores[3] = scores[0], -40.0
    for eos in (0, 5, 2, vocab - 1):
        check(logits, scores, beams, k, finished, eos)
    scores[4] = -np.inf
    check(logits, scores, beams, k, finished, 9)
    check(logits[:, :3].copy(), scores, beams, 6, finished, 2)


def test_beams_whose_scores_lie_close(cuda_lib):
    """Long sums: 32 bits hold steps of 2^-12 there, the order goes by 64."""
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((8, 5000)).astype(np.float32)
    logits[1:] = logits[0] + rng.standard_normal((7, 5000)).astype(np.float32) * np.float32(1e-5)
    check(logits, np.full(8, -30000.0, np.float32), 8, 16)


def test_rows_of_a_wider_buffer(cuda_lib):
    rng = np.random.default_rng(6)
    for offset, width in ((0, 3001), (1, 3004), (4, 3004)):
        wide = rng.standard_normal((6, width + 8)).astype(np.float32)
        d = dev(wide)
        view = wide[:, offset: offset + 2999]
        check(view, np.zeros(6, np.float32), 3, 6, logits_dev=d[:, offset: offset + 2999])


def test_graph_and_side_stream(cuda_lib):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(7)
    a, b = ((rng.standard_normal((4, 40000))).astype(np.float32) for _ in range(2))
    scores = np.zeros(4, np.float32)
    d, s = dev(a), dev(scores)
    kernels.beam_select(d, s, beams=4, k=8)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        for _ in range(2):
            parent, token, _ = kernels.beam_select(d, s, beams=4, k=8, use_pdl=True)
    for x in (a, b, a):
        d.copy_(dev(x))
        graph.replay()
        torch.cuda.synchronize()
        want = ref.select(x, scores, 4, 8)
        assert np.array_equal(host(parent), want[0]) and np.array_equal(host(token), want[1])


@pytest.mark.parametrize("k", [15, 17, 19, 31, 33, 47, 63])
def test_odd_numbers_of_candidates(cuda_lib, k):
    rng = np.random.default_rng(k)
    for beams, vocab in ((32, 1000), (3, 40001), (1, 128256)):
        logits = (rng.standard_normal((2 * beams, vocab)) * 2).astype(np.float32)
        logits[:, ::5] = np.round(logits[:, ::5])
        check(logits, (-9 * rng.random(2 * beams)).astype(np.float32), beams, k)


@pytest.mark.parametrize("beams,vocab,k", [(2, 400000, 64), (1, 1000003, 64), (3, 262144, 33)])
def test_lists_longer_than_a_warp_keeps(cuda_lib, beams, vocab, k):
    rng = np.random.default_rng(vocab)
    logits = (rng.standard_normal((beams, vocab)) * 2).astype(np.float32)
    check(logits, -np.arange(beams, dtype=np.float32), beams, k)
    check(np.round(logits), -np.arange(beams, dtype=np.float32), beams, k)             # the border falls among many alike


def test_many_groups(cuda_lib):
    rng = np.random.default_rng(40)
    logits, scores = rng.standard_normal((3000 * 2, 57)).astype(np.float32), (-5 * rng.random(6000)).astype(np.float32)
    check(logits, scores, 2, 5, finished=(rng.random(6000) < 0.2).astype(np.int32), eos=56)


@pytest.mark.parametrize("grid", [1.0, 0.5, 0.125])
def test_logits_on_a_grid(cuda_lib, grid):
    """Logits of few different values, as those of a coarser type are: errors of their exponentials do not average out."""
    rng = np.random.default_rng(13)
    for spread in (1, 3):
        logits = (np.round(rng.standard_normal((4, 100000)) * spread / grid) * grid).astype(np.float32)
        check(logits, np.arange(4, dtype=np.float32) * -3.3, 2, 64)
    flat = np.full((2, 131072), 0.3, np.float32)                  # as much weight as one token has, 11.4 below it
    flat[:, 7] = 11.7
    check(flat, np.zeros(2, np.float32), 1, 4)


@pytest.mark.parametrize("offset", [3e4, -3e4, 32768, 1e6, -1e9, 1e12, -1e20, 1e36, 2e38, -3e38])
def test_logits_far_from_zero(cuda_lib, offset):
    """Rows that lie around any number, and rows spread as widely: the largest counts for 1, whatever it is."""
    rng = np.random.default_rng(3)
    near = (offset + rng.standard_normal((4, 20000)) * 3).astype(np.float32)
    wide = (rng.standard_normal((4, 20000)) * min(abs(offset), 6e37)).astype(np.float32)
    for logits in (near, wide):
        check(logits, np.array([0, -1, -2, -3], np.float32), 2, 6)


def test_two_at_once(cuda_lib):
    """Calls on two streams, each with a workspace of its own."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(8)
    rows = [(rng.standard_normal((8, 60000)) * 2).astype(np.float32) for _ in range(2)]
    want = [ref.select(x, np.zeros(8, np.float32), 4, 8) for x in rows]
    d, scores, streams = [dev(x) for x in rows], torch.zeros(8, device="cuda"), [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kernels.beam_select(d[i], scores, beams=4, k=8, use_pdl=True))
    torch.cuda.synchronize()
    for i in range(2):
        for parent, token, _ in got[i]:
            assert np.array_equal(host(parent), want[i][0]) and np.array_equal(host(token), want[i][1])


def test_no_groups(cuda_lib):
    from tenzo_b200 import kernels
    parent, token, score = kernels.beam_select(torch.empty(0, 10, device="cuda"), torch.empty(0, device="cuda"), beams=2, k=3)
    assert parent.shape == token.shape == score.shape == (0, 3)


@pytest.mark.parametrize("beams", [1, 4])
@pytest.mark.parametrize("vocab,repeats", [(1000, 1), (8192, 1), (8192, 8), (20001, 3), (128256, 1)])
def test_few_numbers_among_nan(cuda_lib, vocab, repeats, beams):
    """Fewer finite logits than are asked for, at the front, in the middle, at the end and scattered, the rest NaN; NaN and -infinity in turns, at random and by the
    threads that hold them: every finite one counts, then the lowest tokens of those that are masked. (Many rows: as many logits a thread as there can be.)"""
    rng = np.random.default_rng(vocab + beams)
    owner = np.arange(vocab) // 4 % 256
    rests = [np.full(vocab, np.nan), np.where(rng.random(vocab) < 0.5, np.nan, -np.inf), np.where(owner % 2, np.nan, -np.inf), np.where(owner < 200, np.nan, -np.inf)]
    for finite in (0, 1, 12, 15, 17):
        places = [np.arange(finite), vocab // 2 + np.arange(finite), vocab - 1 - np.arange(finite), rng.choice(vocab, finite, replace=False)]
        logits = np.stack([rest for rest in rests for _ in places] * repeats).astype(np.float32)
        for row, at in zip(logits, places * len(rests) * repeats):
            row[at] = np.round(rng.standard_normal(finite) * 8) / 4
        for k in (8, 24):
            check(logits, (-3 * rng.random(len(logits))).astype(np.float32), beams, k)


def test_calls_of_many_and_few_rows_from_two_threads(cuda_lib):
    """The sizes take kernels of their own, whose settings no other thread's call changes; each thread on its stream."""
    import threading
    from tenzo_b200 import kernels
    rng = np.random.default_rng(50)
    logits = [(rng.standard_normal((rows, 16384)) * 2).astype(np.float32) for rows in (512, 64)]              # 1024 chunks, and 128
    want = [ref.select(x, np.zeros(len(x), np.float32), 4, 8) for x in logits]
    d, scores = [dev(x) for x in logits], [torch.zeros(len(x), device="cuda") for x in logits]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got[i].append(kernels.beam_select(d[i], scores[i], beams=4, k=8, use_pdl=True))
        except Exception as e:                           # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for i in range(2):
        for parent, token, _ in got[i]:
            assert np.array_equal(host(parent), want[i][0]) and np.array_equal(host(token), want[i][1])


@pytest.mark.parametrize("groups,beams,vocab,stride,k", [(32, 8, 20004, 20004, 16), (32, 8, 32772, 32772, 5), (64, 4, 20002, 20016, 8), (10, 30, 16387, 16388, 32), (640, 1, 3001, 3004, 4)])
def test_many_chunks_of_aligned_rows(cuda_lib, groups, beams, vocab, stride, k):
    """More CTAs than run at a time, rows that start at 16 bytes: last chunks of a few logits, rows of a wider buffer, vocabularies of any remainder; finished and dead beams, whose rows nothing is
    stored for, over a workspace of NaN."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(vocab)
    wide = (rng.standard_normal((groups * beams, stride)) * 2.5).astype(np.float32)
    wide[:, vocab:] = 1e30                               # (nobody's logits)
    logits = wide[:, :vocab]
    logits[:, 7::911] = -np.inf
    logits[rng.random(logits.shape) < 1e-4] = np.nan
    scores = (-20 - 3 * rng.random(groups * beams)).astype(np.float32)
    scores[rng.random(groups * beams) < 0.05] = -np.inf
    finished = (rng.random(groups * beams) < 0.1).astype(np.int32)
    finished[-2:] = 1                                    # the last rows of the buffer
    d = dev(wide)[:, :vocab]
    got = check(logits, scores, beams, k, finished, 2, logits_dev=d)
    ws = torch.full((kernels.beam_select_workspace_bytes(groups, beams, vocab, k),), 255, dtype=torch.uint8, device="cuda")
    again = kernels.beam_select(d, dev(scores), beams=beams, k=k, finished=dev(finished), eos=2, workspace=ws, use_pdl=True)
    assert all(np.array_equal(x, host(y)) for x, y in zip(got, again))
