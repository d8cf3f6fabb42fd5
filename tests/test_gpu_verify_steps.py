"""Acceptance of drafted tokens where there are too many rows to sum all of them first: a launch per step of all walks, and what is left
of long ones behind them.  Each case also runs with its rows alone, most of them few enough to be summed first."""
import numpy as np
import pytest
import torch

import fstattention_amd as fsta
from fstattention_amd import _lib
from test_gpu_verify import call, cases_of_more_that_fall, check, expected, make_case, on_gpu

pytestmark = pytest.mark.gpu


def by_steps(case):
    """The case on the GPU with rows behind the last sequence, until there are too many to sum all."""
    gpu = on_gpu(case)
    nodes, vocabulary = gpu["logits"].shape
    more = max(int(200e6 / vocabulary) + 1 - nodes, 0)
    pad = lambda t, x: torch.cat([t, torch.full((more, *t.shape[1:]), x, dtype=t.dtype, device="cuda")])
    gpu = {**gpu, "logits": pad(gpu["logits"], 7.0), "tokens": pad(gpu["tokens"], 0), "parent": pad(gpu["parent"], 0), "u_accept": pad(gpu["u_accept"], 0.0),
           "draft_probs": None if gpu["draft_probs"] is None else pad(gpu["draft_probs"], 0.5)}
    # no room for a sum of every row
    work = [_lib.load().fsta_verify_workspace_bytes(1, nodes + more + i, vocabulary, 8, case["draft_probs"] is not None) for i in range(2)]
    assert work[0] == work[1]
    return gpu


def check_both(case, *args, what=""):
    want = expected(case, *args)
    tau = [torch.tensor(a).cuda() if isinstance(a, list) else a for a in args]
    check(call(by_steps(case), *tau), want, what + " by steps")
    check(call(on_gpu(case), *tau), want, what + " alone")


@pytest.mark.parametrize("dtype,draft,vocabulary", [(torch.bfloat16, None, 50021), (torch.float16, torch.float32, 50021), (torch.float32, None, 32000),
                                                    (torch.bfloat16, torch.bfloat16, 131072), (torch.float32, torch.float16, 30011)])
def test_trees(dtype, draft, vocabulary):
    sizes = [1, 30, 0, 64, 17, 90, 2, 45, 80, 64, 100, 33, 64, 200, 64, 64] + [5] * 20
    case = make_case(vocabulary + 1, sizes, vocabulary, dtype, 4, draft)
    check_both(case, 40)
    check_both(case, 3, 0.8, what="cut")
    check_both(case, 12, [0.0, 1.0, 0.5, 1.7] * 9, what="mixed")


@pytest.mark.parametrize("draft", [None, torch.float32])
def test_long_paths(draft):
    """Chains whose tokens are all but certain, longer than there are launches."""
    sizes = [60] * 12 + [7, 1, 0, 40]
    case = make_case(3, sizes, 24001, torch.float32, 1, draft, likely=1.0)
    n = case["tokens"].shape[0]
    starts = case["q_starts"].numpy()
    for b, size in enumerate(sizes):
        s = starts[b]
        for i in range(size):
            case["parent"][s + i] = i - 1
            if i:
                case["logits"][s + i - 1, case["tokens"][s + i]] = 25.0
                if draft is not None:
                    case["draft_probs"][s + i - 1, case["tokens"][s + i]] = 0.5
    assert n == 768
    case["u_accept"][200] = 1.0                                # one falls
    assert expected(case, 64)[1].max() >= 59
    check_both(case, 64)
    check_both(case, 25)


@pytest.mark.parametrize("draft", [None, torch.float32])
def test_many_that_fall(draft):
    """Nodes with a dozen children of which most fall: more sums than launches; little left of a sum, and nothing."""
    sizes = [40] * 30
    case = make_case(6, sizes, 16007, torch.float32, 13, draft, likely=0.0, spread=1.0)
    case["u_accept"][:] = 1.0 - 2.0 ** -24
    rows = case["logits"].view(30, 40, 16007)
    for b in range(10):                                        # the first children have nearly all the mass
        for i in range(1, 4):
            if case["parent"].view(30, 40)[b, i] == 0:
                rows[b, 0, case["tokens"].view(30, 40)[b, i]] = 40.0 - i
    for b in range(10, 15):                                    # the root's children are all there is
        kids = (case["parent"].view(30, 40)[b] == 0).nonzero()[:, 0]
        keep = rows[b, 0, case["tokens"].view(30, 40)[b, kids]].clone()
        rows[b, 0] = -float("inf")
        rows[b, 0, case["tokens"].view(30, 40)[b, kids]] = keep
    case["u_accept"].view(30, 40)[10:13] = 1.0                 # and all of them fall
    check_both(case, 9)
    case["u_accept"][::3] = 0.3
    check_both(case, 9)


@pytest.mark.parametrize("tau", [0.0, 1.0])
@pytest.mark.parametrize("draft", [None, torch.bfloat16])
def test_masked_and_infinite_rows(tau, draft):
    case = make_case(21, [6] * 400, 16000, torch.bfloat16, 2, draft)
    rows = case["logits"].view(400, 6, 16000)
    inf = float("inf")
    rows[0::8] = -inf
    rows[1::8, :, 8195:] = -inf                                # whole parts without anything
    rows[2::8, :, :8192] = float("nan")
    rows[3::8, :, [3, 9000]] = inf
    rows[4::8, :, 15999] = torch.finfo(torch.bfloat16).max
    rows[5::8] = torch.finfo(torch.bfloat16).min
    check_both(case, 6, tau)


@pytest.mark.parametrize("draft", [None, torch.bfloat16])
def test_captured_and_replayed(draft):
    cases = [make_case(s, [64] * 20 + [3] * 10, 30000, torch.bfloat16, 3, draft) for s in (1, 2, 3)]
    held = by_steps(cases[0])
    call(held, 12)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(held, 12)
    for case in cases + cases[:2]:
        for name, t in by_steps(case).items():
            if t is not None:
                held[name].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        check(out, expected(case, 12))
        check(call(held, 12), expected(case, 12))


def test_the_same_answers_by_either_way():
    """A batch too large to sum all its rows, and its halves that are not."""
    sizes = [40] * 32
    case = make_case(12, sizes, 40000, torch.bfloat16, 4, torch.bfloat16)
    whole, gpu = call(by_steps(case), 10), on_gpu(case)
    for b in range(0, 32, 8):
        s = slice(40 * b, 40 * (b + 8))
        part = fsta.verify_drafts(gpu["logits"][s], gpu["tokens"][s], gpu["parent"][s], torch.arange(9, dtype=torch.int32, device="cuda") * 40,
                                  gpu["u_accept"][s], gpu["u_next"][b:b + 8], 10, draft_probs=gpu["draft_probs"][s])
        for a, w in zip(part, whole):
            np.testing.assert_array_equal(a.cpu().numpy(), w[b:b + 8].cpu().numpy())


def test_rows_longer_than_a_part_can_be():
    """A row of more than 256 parts of 8192: parts are longer."""
    vocabulary = 256 * 8192 + 12345
    case = make_case(2, [4, 3, 5, 2], vocabulary, torch.float16, 2, None)
    check_both(case, 5)
    case["logits"][:, 20000:] = -float("inf")
    case["logits"][3, vocabulary - 1] = 30.0
    check_both(case, 5, 0.5)


@pytest.mark.parametrize("tau", [1e-7, 1e-4, 1.0, 1e8])
def test_random_numbers_next_to_what_decides(tau):
    """Random numbers within some 1e-7 of the place where a child stands or falls, or the next token changes: sums in 32 bits do not tell, and
    every answer is that of 64."""
    sizes, vocabulary = [3] * 64, 9001
    case = make_case(77, sizes, vocabulary, torch.float32, 2, None, spread=2.0, likely=0.3)
    case["parent"] = torch.tensor([-1, 0, 0] * 64)
    rows = case["logits"].double()[0::3]
    scaled = (rows - rows.amax(1, keepdim=True)) / float(np.float32(tau))
    p = torch.exp(scaled)
    first = p.gather(1, case["tokens"][1::3, None])[:, 0] / p.sum(1)
    near = torch.linspace(-2e-7, 2e-7, 64, dtype=torch.float64)
    case["u_accept"][1::3] = (first + near).clamp(0, 1).float()
    case["u_accept"][2::3] = 1.0
    case["tokens"][2::3] = case["tokens"][1::3]                # once fallen, it falls
    rest = p.scatter(1, case["tokens"][1::3, None], 0.0)
    run = rest.cumsum(1) / rest.sum(1, keepdim=True)
    case["u_next"] = (run[torch.arange(64), torch.arange(64) * 140] + near).clamp(0, 1).float()
    check_both(case, 2, tau)
    more = make_case(78, [2] * 4000, 3000, torch.float32, 1, None)                            # and where only the last sum counts
    more["logits"][:192] = case["logits"][:, :3000]
    p = torch.exp((more["logits"].double()[0::2] - more["logits"].double()[0::2].amax(1, keepdim=True)) / float(np.float32(tau)))
    run = p.cumsum(1) / p.sum(1, keepdim=True)
    places = torch.arange(4000) % 3000
    more["u_next"] = (run[torch.arange(4000), places] + torch.linspace(-2e-7, 2e-7, 4000, dtype=torch.float64)).clamp(0, 1).float()
    more["u_accept"][:] = 1.0
    check_both(more, 1, tau)


def test_a_large_tree():
    """More nodes than all rows are summed of, whatever they cost."""
    n, vocabulary = 140000, 41
    case = make_case(8, [3], vocabulary, torch.float32, 2, None)
    g = torch.Generator().manual_seed(8)
    case = {**case, "logits": torch.randn((n, vocabulary), generator=g), "tokens": torch.randint(vocabulary, (n,), generator=g),
            "u_accept": torch.rand((n,), generator=g), "q_starts": torch.tensor([0, n], dtype=torch.int32), "u_next": torch.rand((1,), generator=g)}
    case["parent"] = (torch.arange(n) - 1 - (torch.rand((n,), generator=g) * 3000).long()).clamp(min=0)
    case["parent"][0] = -1
    case["logits"][case["parent"][1:], case["tokens"][1:]] = 6.0
    work = [_lib.load().fsta_verify_workspace_bytes(1, n + i, vocabulary, 9, 0) for i in range(2)]
    assert work[0] == work[1]
    want = expected(case, 9)
    assert want[1][0] == 3                                     # the oracle's: nodes 0, 44 and 2255
    check(call(on_gpu(case), 9), want)


@pytest.mark.parametrize("draft", [None, torch.float32])
@pytest.mark.parametrize("vocabulary", [301, 9001])
def test_more_fall_than_there_are_launches(draft, vocabulary):
    for case in cases_of_more_that_fall(draft, vocabulary):
        check_both(case, 3)
