"""fl_verify_device (acceptance and draw of drafted tokens) against the
definition in 64 bits, row by row.

Tokens and counts have to be equal.  The oracle's own sums are in 64 bits in
another order than the kernel's, so a draw within 1e-12 of a border of the
cumulative weights, or an acceptance test within 1e-12 of equality, could
differ; no case here comes that near (asserted).  The acceptance tests use the
kernel's sum of exponentials, which the kernel may take in 32 bits each: 2^-20
relative, so tests nearer than that to equality are asserted away too.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dotnetfoundryllm_b200.paged import PagedBatch, PagedKvCache
from dotnetfoundryllm_b200.runtime import ArgumentError, NotSupportedError, XoshiroRandom
from dotnetfoundryllm_b200.speculate import verify_drafts

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def oracle(logits, starts, draft, temp, u_acc, u_smp, probs=None, near=None):
    """(tokens, accepted); tokens of rows outside every sequence are -7."""
    l = logits.double().cpu().numpy().copy()
    l[np.isnan(l)] = -np.inf
    l = np.minimum(l, np.finfo(np.float32).max)
    rows, V = l.shape
    tokens = np.full(rows, -7, np.int64)
    accepted = []
    for b in range(len(starts) - 1):
        r0, r1 = starts[b], starts[b + 1]
        n, stop, tok = 0, None, -1
        for r in range(r0, r1):
            m, t, d = l[r].max(), float(temp[b]), int(draft[r])
            greedy = not t > 0
            live = m > -np.inf
            e = np.exp((l[r] - m) / (1.0 if greedy else t)) if live else np.zeros(V)
            z = e.sum()
            q = None if probs is None else np.nan_to_num(np.maximum(probs[r].double().cpu().numpy(), 0.0), nan=0.0)
            last = r == r1 - 1
            ok = False
            if not last and live and 0 <= d < V:
                if greedy:
                    ok = d == int(l[r].argmax())
                else:
                    a = float(u_acc[r]) * (1.0 if q is None else q[d]) * z
                    if near is not None and a != e[d]:
                        near.append(abs(a - e[d]) / max(e[d], 1e-300) / 2.0 ** -20)
                    ok = a < e[d]
            if ok:
                tokens[r] = d
                n += 1
                continue
            stop = r
            if live and greedy:
                tok = int(l[r].argmax())
            elif live:
                w = e
                if not last:
                    rest = e.copy()
                    if q is not None:
                        rest = np.maximum(e - q * z, 0.0)
                    elif 0 <= d < V:
                        rest[d] = 0.0
                    if rest.sum() > 0:
                        w = rest
                c = np.cumsum(w)
                goal = float(u_smp[b]) * c[-1]
                tok = int(np.argmax(c > goal))
                if near is not None:
                    near.append(np.abs(c - goal).min() / c[-1] / 1e-12)
            break
        if stop is not None:
            tokens[stop] = tok
            tokens[stop + 1:r1] = -1
        accepted.append(n)
    return tokens, np.array(accepted, np.int64)


def run_case(logits, starts, draft, temp, u_acc, u_smp, probs=None, check_near=True):
    near = []
    want, want_n = oracle(logits, starts, draft, temp, u_acc, u_smp, probs, near)
    if check_near:
        assert all(x > 1 for x in near), "a draw next to a border: take another seed"
    dev = lambda x, t: torch.as_tensor(np.asarray(x), dtype=t).to(DEV)  # noqa: E731
    tokens = torch.full((logits.shape[0],), -7, dtype=torch.int32, device=DEV)
    got, got_n = verify_drafts(logits.to(DEV), dev(starts, torch.int32), dev(draft, torch.int32), dev(temp, torch.float32),
                               dev(u_acc, torch.float32), dev(u_smp, torch.float32),
                               draft_probs=None if probs is None else probs.to(DEV), tokens=tokens)
    np.testing.assert_array_equal(got_n.cpu().numpy(), want_n)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    return want, want_n


def case(seed, V, counts, act=torch.float32, probs=True, flat=False, temps=None):
    g = torch.Generator().manual_seed(seed)
    rows, S = sum(counts), len(counts)
    base = torch.randn(rows, V, generator=g) * (0.01 if flat else 2.0)
    if not flat:
        base.scatter_add_(1, torch.randint(0, V, (rows, 3), generator=g), torch.rand(rows, 3, generator=g) * 8)
    q = torch.softmax(base + 0.4 * torch.randn(rows, V, generator=g), -1)
    draft = torch.multinomial(q, 1, generator=g)[:, 0].numpy()
    temp = torch.rand(S, generator=g).numpy() + np.float32(0.3) if temps is None else np.asarray(temps, np.float32)
    starts = np.concatenate([[0], np.cumsum(counts)])
    return (base.to(act), starts, draft, temp.astype(np.float32), torch.rand(rows, generator=g).numpy(),
            torch.rand(S, generator=g).numpy(), q if probs else None)


@pytest.mark.parametrize("act", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("V", [1, 2, 31, 511, 1000, 4097, 32000, 128256])
def test_matches_the_definition(V, probs, act):
    counts = [1, 5, 0, 3, 8, 2, 9, 1, 4]
    if V > 30000:
        counts = counts[:6]
    run_case(*case(V, V, counts, act, probs and V > 1))


def test_every_outcome_occurs_and_many_sequences():
    seen = set()
    for seed in range(4):
        logits, starts, draft, temp, ua, us, q = case(seed + 50, 257, [seed + 2] * 70)
        _, n = run_case(logits, starts, draft, temp, ua, us, q)
        seen |= set(n.tolist())
    assert {0, 1, 2} <= seen and max(seen) >= 3


@pytest.mark.parametrize("n", [33, 64, 65, 100])
def test_long_drafts(n):
    logits, starts, draft, temp, ua, us, q = case(n, 300, [n, 1, n], temps=[0.7, 0.7, 0.0])
    run_case(logits, starts, draft, temp, ua, us, q)
    # drafts that are all accepted: the bonus token comes from the last row
    top = logits.argmax(1).numpy()
    want, acc = run_case(logits, starts, top, temp, np.zeros_like(ua), us, q)
    assert acc.tolist() == [n - 1, 0, n - 1] and (want >= 0).all()


def test_flat_logits_at_a_large_vocabulary():
    """A nearly uniform target, the cumulative sums' borders close together."""
    run_case(*case(5, 128256, [1, 3, 2, 1], flat=True))
    run_case(*case(6, 128256, [1, 3, 2, 1], act=torch.bfloat16, probs=False, flat=True))


def test_greedy_takes_the_first_maximum():
    logits = torch.zeros(6, 1000)
    logits[0, [5, 700]] = 3.0
    logits[1, [999, 0]] = 2.0
    logits[2, 17] = 1.0
    logits[4, 10] = -0.0
    draft = [5, 999, 17, 3, 0, 0]
    want, n = run_case(logits, [0, 4, 6], draft, [0.0, -1.0], [0.5] * 6, [0.5] * 2)
    assert want.tolist() == [5, 0, -1, -1, 0, 0] and n.tolist() == [1, 1]
    want, n = run_case(logits, [0, 4, 6], draft, [float("nan")] * 2, [0.5] * 6, [0.5] * 2)
    assert n.tolist() == [1, 1]


def test_masked_logits_are_never_accepted_or_drawn():
    V = 5000
    logits, starts, draft, temp, ua, us, q = case(9, V, [4, 3, 2, 2, 3])
    keep = torch.rand(logits.shape, generator=torch.Generator().manual_seed(1)) < 0.01
    keep[0] = False
    keep[0, [3, 4999]] = True
    for low in (-math.inf, float("nan"), torch.finfo(torch.float32).min):
        x = torch.where(keep, logits, torch.full_like(logits, low))
        want, _ = run_case(x, starts, draft, temp, ua, us, q)
        for r, t in enumerate(want):
            assert t < 0 or keep[r, t]
        run_case(x, starts, draft, temp, ua, us, None)


def test_rows_with_nothing_left_and_infinities():
    V = 700
    logits, starts, draft, temp, ua, us, q = case(10, V, [3, 2, 1, 2])
    logits[1] = -math.inf       # stops the first sequence
    logits[3] = float("nan")    # the second sequence's first row
    logits[5] = -math.inf       # the third's only one
    logits[6, 13] = math.inf    # the largest finite: takes all
    ua[0] = 0.0
    want, n = run_case(logits, starts, draft, temp, ua, us, q)
    assert want[3] == -1 and want[4] == -1 and want[5] == -1
    assert n.tolist()[1:3] == [0, 0]
    run_case(logits, starts, draft, [0.0] * 4, ua, us, q)


def test_drafts_outside_the_vocabulary_and_bad_probabilities():
    V = 400
    logits, starts, draft, temp, ua, us, q = case(11, V, [3, 3, 3])
    draft[0], draft[3], draft[6] = -1, V, 2 ** 30
    _, n = run_case(logits, starts, draft, temp, ua, us, q)
    assert n.tolist() == [0, 0, 0]
    run_case(logits, starts, draft, temp, ua, us, None)
    q[:, ::3] = float("nan")
    q[:, 1::3] *= -1.0
    draft = np.full(9, 6)
    run_case(logits, starts, draft, temp, ua, us, q)


def test_a_draft_with_the_targets_own_distribution():
    """q = p up to rounding: rejection is as good as impossible and the rest may be empty."""
    logits, starts, draft, temp, ua, us, _ = case(12, 900, [4, 4], temps=[1.0, 1.0])
    q = torch.softmax(logits.double(), -1).float()
    ua[:] = 0.9999
    run_case(logits, starts, draft, temp, ua, us, q)
    # an impossible draft (certain of a token the target masks) leaves p itself
    logits[0, 5] = -math.inf
    draft[0] = 5
    q[0] = 0.0
    q[0, 5] = 1.0
    _, n = run_case(logits, starts, draft, temp, ua, us, q)
    assert n[0] == 0
    q[0] = 1.0                  # more than p everywhere: nothing is left of p - q
    run_case(logits, starts, draft, temp, ua, us, q)


@pytest.mark.parametrize("u", [0.0, 1 - 2.0 ** -24])
def test_draws_at_the_ends(u):
    logits, starts, draft, temp, _, _, q = case(13, 3001, [2, 1, 3])
    logits[:, 0] = -math.inf
    logits[:, -1] = -math.inf
    for p in (q, None):
        run_case(logits, starts, draft, temp, np.full(6, u, np.float32), np.full(3, u, np.float32), p, check_near=False)


def test_rows_behind_the_last_sequence_are_left_alone():
    logits, starts, draft, temp, ua, us, q = case(14, 300, [2, 3])
    pad = torch.cat([logits, logits])
    want, n = run_case(pad, starts, np.concatenate([draft, draft]), temp, np.concatenate([ua, ua]), us, torch.cat([q, q]))
    assert (want[5:] == -7).all()


def test_strided_rows():
    """Logits inside a wider matrix, rows that start at any element."""
    for off, act in ((0, torch.float32), (1, torch.float16), (3, torch.bfloat16), (1, torch.float32)):
        logits, starts, draft, temp, ua, us, q = case(15, 1003, [3, 4], act)
        wide = torch.full((7, 1011), 50.0, dtype=act, device=DEV)
        wide[:, off:off + 1003] = logits.to(DEV)
        qw = torch.full((7, 1009), 9.0, device=DEV)
        qw[:, 2:1005] = q.to(DEV)
        want, wn = oracle(logits, starts, draft, temp, ua, us, q)
        dev = lambda x, t: torch.as_tensor(np.asarray(x), dtype=t).to(DEV)  # noqa: E731
        got, n = verify_drafts(wide[:, off:off + 1003], dev(starts, torch.int32), dev(draft, torch.int32),
                               dev(temp, torch.float32), dev(ua, torch.float32), dev(us, torch.float32),
                               draft_probs=qw[:, 2:1005])
        np.testing.assert_array_equal(got.cpu().numpy(), want)
        np.testing.assert_array_equal(n.cpu().numpy(), wn)


def test_graph_replay_and_streams():
    logits, starts, draft, temp, ua, us, q = case(16, 5000, [3, 4, 2])
    dev = lambda x, t: torch.as_tensor(np.asarray(x), dtype=t).to(DEV)  # noqa: E731
    args = [logits.to(DEV), dev(starts, torch.int32), dev(draft, torch.int32), dev(temp, torch.float32), dev(ua, torch.float32),
            dev(us, torch.float32)]
    qd = q.to(DEV)
    verify_drafts(*args, draft_probs=qd)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t, n = verify_drafts(*args, draft_probs=qd)
    for seed in range(3):
        logits, starts, draft, temp, ua, us, q = case(20 + seed, 5000, [3, 4, 2])
        for a, b in zip(args, (logits, starts, draft, temp, ua, us)):
            a.copy_(torch.as_tensor(np.asarray(b)))
        qd.copy_(q)
        g.replay()
        want, wn = oracle(logits, starts, draft, temp, ua, us, q)
        np.testing.assert_array_equal(t.cpu().numpy(), want)
        np.testing.assert_array_equal(n.cpu().numpy(), wn)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(verify_drafts(*args, draft_probs=qd))
    torch.cuda.synchronize()
    for t2, n2 in outs:
        np.testing.assert_array_equal(t2.cpu().numpy(), want)


def test_the_accepted_and_drawn_tokens_follow_the_target():
    """Speculative sampling leaves the target's distribution unchanged: the first
    token's frequencies over many draws, against p by a chi-square bound."""
    V, S = 12, 40000
    g = torch.Generator().manual_seed(3)
    one, qone = torch.randn(1, V, generator=g), torch.softmax(torch.randn(1, V, generator=g), -1)
    logits = one.expand(2 * S, V).contiguous().to(DEV)
    q = qone.expand(2 * S, V).contiguous().to(DEV)
    draft = torch.multinomial(qone[0], 2 * S, replacement=True, generator=g).to(torch.int32).to(DEV)
    starts = torch.arange(0, 2 * S + 1, 2, dtype=torch.int32, device=DEV)
    tok, _ = verify_drafts(logits, starts, draft, torch.ones(S, device=DEV), torch.rand(2 * S, generator=g).to(DEV),
                           torch.rand(S, generator=g).to(DEV), draft_probs=q)
    first = torch.bincount(tok[::2].long().cpu(), minlength=V).double()
    p = torch.softmax(one[0].double(), -1)
    chi2 = ((first - S * p) ** 2 / (S * p)).sum().item()
    assert chi2 < 11 + 6 * math.sqrt(22)   # mean and six standard deviations of chi-square with 11 degrees of freedom


def test_refusals_of_tensors():
    f = lambda *s: torch.zeros(*s, device=DEV)                       # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)    # noqa: E731
    good = dict(logits=f(4, 10), row_start=i(3), draft=i(4), temperature=f(2), u_accept=f(4), u_sample=f(2))
    verify_drafts(**good)
    for over in (dict(draft=i(3)), dict(draft=f(4)), dict(row_start=f(3)), dict(temperature=f(3)), dict(u_accept=f(2)),
                 dict(u_sample=i(2)), dict(logits=f(4, 10).cpu()), dict(logits=f(10, 4).T), dict(draft_probs=f(4, 9)),
                 dict(draft_probs=f(4, 10).half()), dict(tokens=i(3)), dict(row_start=i(0))):
        with pytest.raises(ArgumentError):
            verify_drafts(**{**good, **over})
    with pytest.raises(NotSupportedError):
        verify_drafts(**{**good, "logits": f(4, 10).double()})


# ── the operators together ──────────────────────────────────────────────────
class ToyTarget:
    """One attention layer over a paged cache with tied embeddings, enough for
    greedy decoding to depend on every cached position."""

    def __init__(self, kv, page=16, hd=64, n_kv=2, group=2, vocab=997, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=DEV)      # noqa: E731
        h = hd * n_kv * group
        self.hd, self.n_kv, self.heads, self.vocab = hd, n_kv, n_kv * group, vocab
        self.emb, self.wq = r(vocab, h), r(h, self.heads * hd) / math.sqrt(h)
        self.wkv, self.wo = r(h, 2 * n_kv * hd) / math.sqrt(h), r(self.heads * hd, h) / math.sqrt(h)
        self.cache = PagedKvCache.empty(24, page, n_kv, hd, kv, DEV)
        self.pos = r(400, h) * 0.5

    def step(self, tokens, positions, batch):
        x = self.emb[tokens] + self.pos[positions]
        n = len(tokens)
        kv = (x @ self.wkv).view(n, 2 * self.n_kv, self.hd)
        self.cache.append(batch, kv[:, :self.n_kv], kv[:, self.n_kv:])
        o = self.cache.attention(batch, (x @ self.wq).view(n, self.heads, self.hd), 1 / math.sqrt(self.hd))
        return (x + o.view(n, -1) @ self.wo) @ self.emb.T


@pytest.mark.parametrize("kv", [torch.float16, torch.int8, torch.float8_e4m3fn])
def test_speculative_decoding_gives_the_tokens_of_plain_decoding(kv):
    """Two sequences, drafts that are sometimes right: append, attend, verify,
    and rewind by the length alone, against one token at a time."""
    prompts = [[5, 9, 200, 31, 7], [800, 3]]
    n_new, n_draft = 40, 4
    table = torch.randperm(24, generator=torch.Generator().manual_seed(1))[:2 * 8].view(2, 8).to(torch.int32).to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731

    def feed(model, per_seq, lens):
        """Feeds per_seq[b] tokens at the end of lens[b]; the rows' logits."""
        counts = [len(t) for t in per_seq]
        starts = [0, counts[0], sum(counts)]
        batch = PagedBatch(table, i32([a + c for a, c in zip(lens, counts)]), i32(starts), max_rows=max(counts))
        pos = [a + j for a, c in zip(lens, counts) for j in range(c)]
        return model.step(torch.tensor(sum(per_seq, []), device=DEV), torch.tensor(pos, device=DEV), batch), starts

    plain = ToyTarget(kv)
    logits, starts = feed(plain, [p[:] for p in prompts], [0, 0])
    seqs, lens = [p[:] for p in prompts], [len(p) for p in prompts]
    nxt = [int(logits[s - 1].argmax()) for s in starts[1:]]
    for _ in range(n_new):
        for b in range(2):
            seqs[b].append(nxt[b])
        logits, _ = feed(plain, [[t] for t in nxt], lens)
        lens = [n + 1 for n in lens]
        nxt = [int(t) for t in logits.argmax(1)]

    spec = ToyTarget(kv)
    feed(spec, [p[:-1] for p in prompts], [0, 0])
    got, rng, steps = [p[:] for p in prompts], XoshiroRandom(7), 0
    while min(len(g) - len(p) for g, p in zip(got, prompts)) < n_new:
        drafts = []
        for b in range(2):
            truth = seqs[b][len(got[b]):len(got[b]) + n_draft]
            truth += [1] * (n_draft - len(truth))
            drafts.append([t if rng.next_float() < 0.7 else int(rng.next_float() * 997) for t in truth])
        fed = [[got[b][-1]] + drafts[b] for b in range(2)]
        logits, starts = feed(spec, fed, [len(g) - 1 for g in got])
        rows = starts[-1]
        draft = i32(sum((d + [-1] for d in drafts), []))
        tok, acc = verify_drafts(logits, i32(starts), draft, torch.zeros(2, device=DEV), torch.zeros(rows, device=DEV),
                                 torch.zeros(2, device=DEV))
        tok, acc = tok.tolist(), acc.tolist()
        for b in range(2):
            got[b] += tok[starts[b]:starts[b] + acc[b] + 1]
        steps += 1
    for g, s in zip(got, seqs):
        n = min(len(g), len(s))
        assert g[:n] == s[:n]
    assert steps < n_new   # drafts were accepted
