"""Acceptance of drafted tokens (verify_drafts) against its definition in 64 bits on the host.  Answers are whole numbers and have
to be equal: both sides take their sums in 64 bits, off by some 1e-13 of them, so that one of the few thousand random numbers here falls
between the two with a chance below 1e-6."""
import math
import random

import numpy as np
import pytest
import torch

import fstattention_amd as fsta
from decoding_oracle import verify

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def make_trees(rng, sizes, children):
    """Random trees: parents within each tree, numbered from its root."""
    parent = []
    for n in sizes:
        count, up = [0] * max(n, 1), []
        for i in range(n):
            room = [j for j in range(i) if count[j] < children]
            p = rng.choice(room[-4:] if rng.random() < 0.7 else room) if room and i else -1
            if p >= 0:
                count[p] += 1
            up.append(p)
        parent += up
    return np.array(parent, dtype=np.int64), np.cumsum([0] + list(sizes)).astype(np.int32)


def make_case(seed, sizes, vocabulary, dtype, children=3, draft_dtype=None, spread=3.0, pad=0, likely=0.6):
    """Logits whose most likely tokens are the children's, drafts drawn one after the other without putting back."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    parent, starts = make_trees(rng, sizes, children)
    total = int(starts[-1])
    logits = (torch.randn((total, vocabulary + pad), generator=g) * spread).to(dtype)[:, :vocabulary]
    tokens = torch.randint(vocabulary, (total,), generator=g)
    first = np.repeat(starts[:-1], np.diff(starts))
    draft = None
    if draft_dtype is not None:
        draft = torch.softmax(logits.float() + torch.randn((total, vocabulary), generator=g), -1).to(draft_dtype)
    drawn = {}
    for t in range(total):
        if parent[t] < 0:
            continue
        up = int(first[t] + parent[t])
        if draft is not None:
            seen = drawn.setdefault(up, [])
            q = draft[up].double().clone()
            q[seen] = 0
            if q.sum() > 0:
                tokens[t] = int(torch.multinomial(q, 1, generator=g))
            seen.append(int(tokens[t]))
        elif rng.random() < likely:
            logits[up, tokens[t]] = logits[up].max() + 1.0
    return dict(logits=logits, tokens=tokens, parent=torch.from_numpy(parent), q_starts=torch.from_numpy(starts), draft_probs=draft,
                u_accept=torch.rand((total,), generator=g), u_next=torch.rand((len(sizes),), generator=g))


def on_gpu(case):
    gpu = {k: None if v is None else v.cuda() for k, v in case.items()}
    if not case["logits"].is_contiguous():                    # .cuda() would keep no padding
        whole = torch.zeros((case["logits"].shape[0], case["logits"].stride(0)), dtype=case["logits"].dtype, device="cuda")
        gpu["logits"] = whole[:, :case["logits"].shape[1]].copy_(case["logits"])
    return gpu


def call(gpu, max_path, temperature=1.0, **changes):
    gpu = {**gpu, **changes}
    return fsta.verify_drafts(gpu["logits"], gpu["tokens"], gpu["parent"], gpu["q_starts"], gpu["u_accept"], gpu["u_next"], max_path,
                              temperature=temperature, draft_probs=gpu["draft_probs"])


def expected(case, max_path, temperature=1.0):
    batch = len(case["q_starts"]) - 1
    tau = np.asarray(temperature, dtype=np.float32).astype(np.float64) * np.ones(batch)
    return verify(case["logits"].double().numpy(), case["tokens"].numpy(), case["parent"].numpy(), case["q_starts"].numpy(),
                  case["u_accept"].double().numpy(), case["u_next"].double().numpy(), tau,
                  None if case["draft_probs"] is None else case["draft_probs"].double().numpy(), max_path)


def check(got, want, what=""):
    for name, a, b in zip(("path", "counts", "next_tokens"), got, want):
        np.testing.assert_array_equal(a.cpu().numpy(), b, err_msg=f"{what} {name}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("draft", [None, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocabulary", [1, 2, 7, 8, 9, 130, 511, 1000, 4097, 8193])
def test_trees(dtype, draft, vocabulary):
    children = min(3, vocabulary)
    case = make_case(vocabulary + 17, [1, 9, 0, 24, 5, 2, 40], vocabulary, dtype, children, draft, pad=3)
    check(call(on_gpu(case), 12), expected(case, 12))
    check(call(on_gpu(case), 2), expected(case, 2), "cut")
    check(call(on_gpu(case), 1, 0.7), expected(case, 1, 0.7), "roots only")


@pytest.mark.parametrize("dtype,draft,vocabulary", [(torch.bfloat16, None, 131072), (torch.float32, None, 100003), (torch.float16, torch.float16, 50021),
                                                    (torch.bfloat16, torch.float32, 32000), (torch.float32, torch.bfloat16, 131071)])
def test_large_vocabularies(dtype, draft, vocabulary):
    case = make_case(vocabulary, [7, 12, 3], vocabulary, dtype, 3, draft, pad=0 if vocabulary % 2 else 5)
    check(call(on_gpu(case), 8, 0.9), expected(case, 8, 0.9))


@pytest.mark.parametrize("draft", [None, torch.float32])
def test_temperatures_of_a_batch(draft):
    sizes = [11, 20, 3, 15, 9, 17, 1, 30]
    case = make_case(5, sizes, 3001, torch.bfloat16, 4, draft)
    tau = [0.0, 1.0, 0.3, 2.5, -1.0, 1e-3, 1e6, 1e-30]
    gpu = on_gpu(case)
    check(call(gpu, 9, torch.tensor(tau).cuda()), expected(case, 9, tau))
    assert not torch.equal(call(gpu, 9, 0.0).next_tokens, call(gpu, 9, 2.0).next_tokens)
    check(call(gpu, 9, 0.0), expected(case, 9, 0.0))
    check(call(gpu, 9, 0), expected(case, 9, 0.0), "a whole number")
    inf = torch.tensor([float("nan"), float("inf")] * 4).cuda()
    check(call(gpu, 9, inf), expected(case, 9, [float("nan"), float("inf")] * 4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("draft", [None, torch.float32])
@pytest.mark.parametrize("tau", [0.0, 1.0])
def test_masked_infinite_and_nan_logits(dtype, draft, tau):
    case = make_case(21, [6] * 9, 700, dtype, 2, draft)
    rows = case["logits"].view(9, 6, 700)
    rows[0] = -math.inf                                        # nothing may be chosen
    rows[1, :, 5:] = -math.inf                                 # a few tokens may
    rows[2, :, ::3] = math.nan
    rows[3, :, [3, 90]] = math.inf
    rows[4] = math.nan
    rows[5] = torch.finfo(dtype).min                           # as good as any other value
    rows[6, 0] = -math.inf                                     # only the root's
    rows[7, 1:] = -math.inf                                    # all but the root's
    rows[8, :, 699] = torch.finfo(dtype).max
    check(call(on_gpu(case), 6, tau), expected(case, 6, tau))
    gpu = on_gpu(case)
    assert gpu["logits"].isnan().any() and call(gpu, 6, tau).next_tokens[0] == -1


@pytest.mark.parametrize("draft", [None, torch.float16])
@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, math.nan])
def test_random_numbers_at_and_past_their_range(draft, u):
    case = make_case(33, [8, 8, 8, 1], 999, torch.float32, 3, draft)
    case["u_next"][:] = u
    check(call(on_gpu(case), 9), expected(case, 9))
    case["u_accept"][:] = u
    check(call(on_gpu(case), 9), expected(case, 9))


@pytest.mark.parametrize("draft", [None, torch.float32])
def test_tokens_and_parents_that_are_none(draft):
    """Tokens outside the vocabulary and tokens asked twice fall; parents that are none lead nowhere; children are asked in order."""
    for seed in range(6):
        case = make_case(seed, [30, 25, 2], 50, torch.float32, 6, draft)
        r = random.Random(seed)
        for _ in range(6):
            case["tokens"][r.randrange(57)] = r.choice([-1, 50, 1 << 40, -(1 << 62), 2 ** 32])
            a = r.randrange(1, 57)
            case["tokens"][a] = case["tokens"][a - 1]
            case["parent"][r.randrange(57)] = r.choice([-7, 29, 1 << 33, 1000])
        case["parent"][0] = 5                                  # a root is the root whatever its own entry says
        check(call(on_gpu(case), 20), expected(case, 20), f"seed {seed}")


def test_draft_that_knows_some_tokens_only():
    """Rows of the draft with zeros, negative values and NaN, and rows without any mass: a child without a probability is taken for a
    given one."""
    case = make_case(8, [20, 20, 20], 64, torch.float32, 6, torch.float32)
    g = torch.Generator().manual_seed(1)
    case["draft_probs"][torch.rand((60, 64), generator=g) < 0.4] = 0
    case["draft_probs"][20:25] = 0
    case["draft_probs"][3] = -1.0
    case["draft_probs"][5, ::2] = math.nan
    case["draft_probs"][40] = 0
    case["draft_probs"][40, 7] = 1.0                           # all mass at one token
    check(call(on_gpu(case), 20), expected(case, 20))


def test_starts_that_leave_nodes_out_and_point_outside():
    case = make_case(9, [6, 7, 8], 100, torch.float16, 2)
    for starts in ([2, 6, 13, 19], [0, 0, 13, 21], [-5, 6, 13, 400], [6, 6, 6, 6], [30, 40, 50, 60]):
        case["q_starts"] = torch.tensor(starts, dtype=torch.int32)
        case["parent"] = torch.tensor([-1] + [0] * 20)
        check(call(on_gpu(case), 5), expected(case, 5), str(starts))


def test_many_children():
    """More children of one node than are asked, and more than one strip of nodes; a token behind all of them."""
    n = 2500
    case = make_case(3, [n], 6000, torch.float32, 1)
    case["parent"] = torch.tensor([-1] + [0] * (n - 1))
    case["tokens"] = torch.arange(n) * 2
    case["logits"][0, ::2] -= 60.0                             # (hardly anything) for the children
    assert call(on_gpu(case), 4).counts.item() == 1
    check(call(on_gpu(case), 4), expected(case, 4))
    case["u_accept"][:] = 1.0
    case["u_accept"][n - 1] = -1.0                             # would be taken if it were asked: it is the 2499th
    assert call(on_gpu(case), 4).counts.item() == 1
    case["u_accept"][2048] = -1.0                              # the 2048th
    assert call(on_gpu(case), 4).path[0].tolist() == [0, 2048, -1, -1]


@pytest.mark.parametrize("shift", range(0, 8))
def test_rows_at_any_address(shift):
    case = make_case(40, [9, 9], 1001, torch.float16, 3, torch.float16)
    gpu = on_gpu(case)
    for name in ("logits", "draft_probs"):
        flat = torch.zeros(18 * 1001 + 16, dtype=torch.float16, device="cuda")
        gpu[name] = flat[shift:shift + 18 * 1001].view(18, 1001).copy_(gpu[name])
    check(call(gpu, 9), expected(case, 9))


def test_rows_repeated_and_one_row_only():
    """A stride of 0 (one row for all nodes), and views with one node."""
    case = make_case(41, [5, 5], 300, torch.float32, 2)
    case["logits"] = case["logits"][:1].expand(10, 300).contiguous()
    gpu = on_gpu(case)
    check(call(gpu, 5, logits=gpu["logits"][:1].expand(10, 300)), expected(case, 5))
    one = make_case(42, [1], 300, torch.float32)
    check(call(on_gpu(one), 5), expected(one, 5))


def test_far_rows():
    """Rows behind the 2^32nd element."""
    vocabulary, rows = 131072, 33000
    logits = torch.full((rows, vocabulary), -2.0, dtype=torch.bfloat16, device="cuda")
    assert logits.numel() > 2 ** 32
    starts = torch.tensor([0, 2, rows - 3, rows], dtype=torch.int32, device="cuda")
    parent = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    parent[rows - 2], parent[rows - 1], parent[1] = 0, 1, 0
    tokens = torch.full((rows,), 9, dtype=torch.int64, device="cuda")
    logits[rows - 3, 9] = 60.0
    logits[rows - 2, 9] = 60.0
    logits[rows - 1, 100001] = 60.0
    u = torch.full((rows,), 0.5, device="cuda")
    got = fsta.verify_drafts(logits, tokens, parent, starts, u, u[:3], 4)
    assert got.path[2].tolist() == [0, 1, 2, -1] and got.next_tokens[2].item() == 100001 and got.counts.tolist() == [1, 1, 3]
    assert got.next_tokens[0].item() == vocabulary // 2 - 1 or got.next_tokens[0].item() == vocabulary // 2


@pytest.mark.parametrize("draft", [False, True])
def test_the_longest_rows(draft):
    """Rows of as many tokens as there may be, whose parts' ends pass 31 bits; three of them have weight."""
    vocabulary, middle = 2 ** 31 - 1 - 65536, 2 ** 30 + 3
    row = torch.full((1, vocabulary), -math.inf, dtype=torch.float16, device="cuda")
    row[0, [5, middle, vocabulary - 1]] = 0.5
    drafts = torch.zeros((1, vocabulary), dtype=torch.float16, device="cuda") if draft else None
    if draft:
        drafts[0, middle] = 1.0
    for u, u_next, path, following in ((0.9, 0.75, [0, -1], vocabulary - 1), (0.9, 0.25, [0, -1], 5), (0.2, 0.99, [0, 1], vocabulary - 1), (0.2, 0.5, [0, 1], middle)):
        got = fsta.verify_drafts(row.expand(2, -1), torch.tensor([0, middle]).cuda(), torch.tensor([-1, 0]).cuda(), torch.tensor([0, 2]).int().cuda(),
                                 torch.tensor([0.0, u]).cuda(), torch.tensor([u_next]).cuda(), 2, draft_probs=drafts.expand(2, -1) if draft else None)
        assert got.path.tolist() == [path] and got.next_tokens.tolist() == [following]


@pytest.mark.parametrize("draft", [False, True])
def test_answers_are_distributed_as_the_models_own(draft):
    """What stands behind the root is a sample of the model's own distribution, whatever was drafted: 200000 trees of up to three children,
    Pearson's statistic over 12 tokens (11 degrees of freedom) below 46 (1 - chi2.cdf = 3e-6; the seed is fixed)."""
    batch, vocabulary = 200000, 12
    g = torch.Generator(device="cuda").manual_seed(11)
    row = torch.randn(vocabulary, generator=g, device="cuda") * 1.5
    q = torch.softmax(row + torch.randn(vocabulary, generator=g, device="cuda"), 0)
    parent = torch.tensor([-1, 0, 0, 0]).repeat(batch).cuda()
    race = q / torch.empty((batch, vocabulary), device="cuda").exponential_(generator=g)
    children = race.topk(3, -1).indices if draft else torch.tensor([7, 2, 5]).cuda().expand(batch, 3)
    tokens = torch.cat([torch.zeros((batch, 1), dtype=torch.int64, device="cuda"), children], 1).reshape(-1)
    starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * 4
    got = fsta.verify_drafts(row.expand(4 * batch, vocabulary), tokens, parent, starts, torch.rand(4 * batch, generator=g, device="cuda"),
                             torch.rand(batch, generator=g, device="cuda"), 2, draft_probs=q.expand(4 * batch, vocabulary) if draft else None)
    accepted = got.path[:, 1].long()
    said = torch.where(accepted >= 0, tokens.view(batch, 4).gather(1, accepted.clamp(min=0)[:, None])[:, 0], got.next_tokens)
    seen = torch.bincount(said, minlength=vocabulary).double()
    want = torch.softmax(row.double(), 0) * batch
    assert float(((seen - want) ** 2 / want).sum()) < 46
    assert 0.2 < (accepted >= 0).double().mean().item() < 0.999


def test_a_sequence_alone_and_in_a_batch():
    sizes = [9, 30, 2, 14] * 40
    case = make_case(70, sizes, 2000, torch.bfloat16, 3, torch.bfloat16)
    gpu = on_gpu(case)
    got = call(gpu, 10)
    check(got, expected(case, 10))
    for b in (0, 1, 2, 3, 77, 159):
        s = slice(int(case["q_starts"][b]), int(case["q_starts"][b + 1]))
        alone = fsta.verify_drafts(gpu["logits"][s], gpu["tokens"][s], gpu["parent"][s], torch.tensor([0, s.stop - s.start], dtype=torch.int32).cuda(),
                                   gpu["u_accept"][s], gpu["u_next"][b:b + 1], 10, draft_probs=gpu["draft_probs"][s])
        for a, w in zip(alone, got):
            assert torch.equal(a[0], w[b])


def test_captured_and_replayed():
    """New logits, tokens and random numbers in the same tensors, with eager calls between the replays."""
    cases = [make_case(s, [9, 16, 4], 3000, torch.bfloat16, 3, torch.float32) for s in (1, 2, 3)]
    held = on_gpu(cases[0])
    call(held, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(held, 8)
    for case in cases + cases[:2]:
        for name, t in on_gpu(case).items():
            held[name].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        check(out, expected(case, 8))
        check(call(held, 8), expected(case, 8))


def test_two_streams_at_once():
    cases = [make_case(s, [16] * 24, 20000, torch.float16, 3, torch.float16 if s else None) for s in (0, 1)]
    gpus = [on_gpu(c) for c in cases]
    wants = [expected(c, 9) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(call(gpus[i], 9))
    torch.cuda.synchronize()
    for i in range(2):
        for got in outs[i]:
            check(got, wants[i])


def test_logits_that_require_a_gradient():
    """Whole numbers have no derivative: as argmax, the call takes them."""
    case = make_case(4, [5, 6], 100, torch.float32, 2)
    gpu = on_gpu(case)
    check(call(gpu, 4, logits=gpu["logits"].clone().requires_grad_()), expected(case, 4))
    with torch.inference_mode():
        check(call(gpu, 4), expected(case, 4))


def test_refusals():
    case = on_gpu(make_case(1, [5, 6], 100, torch.float32, 2, torch.float32))
    for change, word in ((dict(logits=case["logits"].double()), "float32"), (dict(logits=case["logits"][0]), "vocabulary"),
                         (dict(logits=case["logits"].t().contiguous().t()), "contiguous"), (dict(logits=case["logits"][:, :0]), "vocabulary"),
                         (dict(tokens=case["tokens"].int()), "tokens"), (dict(tokens=case["tokens"][:5]), "tokens"), (dict(parent=case["parent"].int()), "parent"),
                         (dict(parent=case["parent"].cpu()), "parent"), (dict(q_starts=case["q_starts"].long()), "q_starts"),
                         (dict(q_starts=case["q_starts"][:0]), "q_starts"), (dict(u_accept=case["u_accept"].double()), "u_accept"),
                         (dict(u_next=case["u_next"][:1]), "u_next"), (dict(u_accept=case["u_accept"].repeat(2)[::2]), "u_accept"),
                         (dict(draft_probs=case["draft_probs"][:, :50]), "draft_probs"), (dict(draft_probs=case["draft_probs"].cpu()), "device"),
                         (dict(draft_probs=case["draft_probs"].double()), "draft_probs")):
        with pytest.raises(ValueError, match=word):
            call(case, 4, **change)
    for temperature in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="temperature"):
            call(case, 4, temperature)
    with pytest.raises(ValueError, match="temperature"):
        call(case, 4, torch.ones(3).cuda())
    with pytest.raises(ValueError, match="max_path"):
        call(case, 0)


def test_no_sequences_and_no_nodes():
    case = on_gpu(make_case(1, [5], 100, torch.float32, 2))
    got = call(case, 4, q_starts=case["q_starts"][:1], u_next=case["u_next"][:0])
    assert got.path.shape == (0, 4) and got.counts.shape == (0,)
    none = {k: v[:0] for k, v in case.items() if v is not None and k not in ("q_starts", "u_next")}
    got = call({**case, **none}, 4, q_starts=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert got.counts.tolist() == [0] and got.next_tokens.tolist() == [-1] and got.path.tolist() == [[-1] * 4]


@pytest.mark.parametrize("draft", [None, torch.float32])
def test_a_token_with_nearly_all_mass_falls(draft):
    """The sum without it is taken again, wherever in the row it stands."""
    vocabulary = 24001
    places = list(range(20)) + [31, 32, 63, 504, 511, 512, 1023, 1024, 1500, 2047, 2048, 5000, 9999, 10000, 20479, 20480, 23551, 23552, 23992, 23993, 24000]
    n = len(places)
    case = make_case(5, [2] * n, vocabulary, torch.float32, 1, None, spread=1.0)
    case["parent"] = torch.tensor([-1, 0] * n)
    case["tokens"] = torch.tensor([t for x in places for t in (0, x)])
    case["logits"][torch.arange(0, 2 * n, 2), torch.tensor(places)] = 25.0
    case["u_accept"][:] = 1.0                                  # it falls all the same
    if draft is not None:
        case["draft_probs"] = torch.zeros((2 * n, vocabulary))
    check(call(on_gpu(case), 3), expected(case, 3))


def cases_of_more_that_fall(draft, vocabulary):
    """Twenty children of one node, drawn or given, of which any number falls; the ones behind those that fell are asked as well."""
    n = 40
    case = make_case(9, [21] * n, vocabulary, torch.float32, 20, None, spread=1.5)
    case["parent"] = torch.tensor(([-1] + [0] * 20) * n)
    g = torch.Generator().manual_seed(4)
    case["tokens"] = torch.stack([torch.randperm(vocabulary, generator=g)[:21] for _ in range(n)]).reshape(-1)
    if draft is not None:
        case["draft_probs"] = torch.softmax(case["logits"] + torch.randn((21 * n, vocabulary), generator=g), -1)
    else:                                                      # the first ones have all but a thousandth of what is left, each
        rows = case["logits"].view(n, 21, vocabulary)
        for b in range(n):
            for i in range(1, 1 + b % 6):
                rows[b, 0, case["tokens"].view(n, 21)[b, i]] = 70.0 - 10.0 * i
    u = case["u_accept"].view(n, 21)
    u[:] = 1.0 - 2.0 ** -24
    for b in range(n):
        u[b, 1 + b % 20] = 0.0                                 # stands, if anything is left of it
    yield case
    u[:] = 1.0 - 2.0 ** -24
    yield case


@pytest.mark.parametrize("draft", [None, torch.float32])
@pytest.mark.parametrize("vocabulary", [40, 3000])
def test_more_fall_than_there_are_launches(draft, vocabulary):
    for case in cases_of_more_that_fall(draft, vocabulary):
        check(call(on_gpu(case), 3), expected(case, 3))
