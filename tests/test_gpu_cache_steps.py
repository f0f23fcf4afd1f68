"""Decode steps over shared prefixes and over caches that are cut down, all operators
together."""
import math

import pytest
import torch

from linuxnightmaresuite_b200 import attention, kernels as K
from linuxnightmaresuite_b200.attention import PagedKVCache

from ._attention import BF16, E4M3, F16, SCALES, attend, rotate
from .test_gpu_attention import _decoder, randn
from .test_gpu_cache_weights import evict_plain, i32, normed, weights

pytestmark = pytest.mark.gpu


def normed_decoder(dtype, qtype=2, gemma=True):
    stack, mats = _decoder(dtype, qtype)
    for i, a in enumerate(stack.attention):
        a.q_norm, a.k_norm = (0.2 * randn(64, seed=7 + i + s) + (0.0 if gemma else 1.0)
                              for s in (0, 1))
        a.gemma_style, a.norm_eps = gemma, 1e-5
    return stack, mats


@pytest.mark.parametrize("dtype,S,tokens", [(F16, 64, 8192), (BF16, 5, 128), (E4M3, 64, 16384)])
def test_steps_behind_a_shared_prompt(dtype, S, tokens):
    """Sequences that share a prompt's pages against 64 bits and, through the stack, against
    the layers one by one; the prompt enters as keys and values of the host's own prefill."""
    hkv, d, page = 2, 64, 64
    ks, vs = SCALES[dtype]
    stack, mats = normed_decoder(dtype)
    width = tokens // page + 1
    caches = [PagedKVCache(width + S + 3, page, hkv, d, S + 1, width, dtype, ks, vs) for _ in range(2)]
    for li, c in enumerate(caches):
        c.reserve(S, tokens)                        # the prompt is a sequence of its own
        k, v = randn(tokens, hkv, d, seed=li), randn(tokens, hkv, d, seed=5 + li)
        c.append(None, k, v, torch.arange(tokens, dtype=torch.int32, device="cuda"),
                 seq_ids=torch.full((tokens,), S, dtype=torch.int32, device="cuda"))
        for s in range(S):
            c.share(s, S, tokens)
        assert c.free_pages == S + 4
    freq = K.rope_inv_freq(d)
    for step in range(3):
        own = [-1 if (s + step) % 5 == 4 else step for s in range(S)]
        pos = [tokens + n if n >= 0 else -1 for n in own]
        for c in caches:
            for s, p in enumerate(pos):
                c.reserve(s, p + 1)
        positions, lens = i32(*pos), i32(*(p + 1 for p in pos))
        x = randn(S, 512, seed=30 + step)
        kw = dict(positions=positions, seq_lens=lens, max_len=tokens + 3)
        before = [(c.k.clone(), c.v.clone()) for c in caches]
        y = stack.forward(x, caches=caches, prefixes=[c.prefix(S, tokens) for c in caches], **kw)
        for c, (k, v) in zip(caches, before):
            c.k.copy_(k), c.v.copy_(v)
        cur = x
        for i, c in enumerate(caches):
            xn = K.rms_norm(cur, stack.attention_norms[i], stack.eps)
            nxt = stack.attention[i].forward(xn, c, positions, lens, residual=cur,
                                             max_len=tokens + 3, prefix=c.prefix(S, tokens))
            wq, _, _, wo = mats[i]
            for s in range(0, S, 7):
                if pos[s] < 0:
                    assert torch.equal(nxt[s], cur[s])
                    continue
                a = stack.attention[i]
                q, _ = normed((wq @ xn[s].double()).view(1, 8, d), a.q_norm, a.norm_eps, True)
                q, _ = rotate(q, positions[s:s + 1], freq, False)
                t = torch.arange(pos[s] + 1, device="cuda")
                pages = c.block_table[s][t // page].long()
                kd, vd = c.k[pages, t % page].double() * ks, c.v[pages, t % page].double() * vs
                o, _, to, _ = attend(q[0], kd, vd, d ** -0.5)
                want = wo @ o.reshape(-1) + cur[s].double()
                # the projection, norm and rotation of q are f32; two parts of a bf16 probability
                tol = wo.abs() @ (to + 2.0 ** -15 * vd.abs().amax()).reshape(-1) + 1e-5
                assert ((nxt[s].double() - want).abs() <= tol).all(), (step, i, s)
            cur = stack.layers[i].forward_batch(K.rms_norm(nxt, stack.norms[i], stack.eps),
                                                residual=nxt)
        assert torch.equal(cur, y)
    for c in caches:
        assert c.device_status() == 0
    for a in stack.attention:
        assert a.device_status() == 0


@pytest.mark.parametrize("dtype,keep,every", [(F16, 12, 1), (BF16, 20, 9), (E4M3, 8, 3)])
def test_steps_over_a_cache_that_is_cut(dtype, keep, every):
    """Sequences decode past `keep` tokens; every few steps all layers give up what has been
    attended to least.  Ledgers and caches against plain forms on the step's own inputs."""
    hkv, hq, d, S, page, recent, steps = 2, 8, 64, 3, 4, 4, 40
    ks, vs = SCALES[dtype]
    stack, mats = normed_decoder(dtype, gemma=False)
    caches = [PagedKVCache(40, page, hkv, d, S, 10, dtype, ks, vs, track=True) for _ in range(2)]
    first = [0, 3, 7]                               # sequences join
    n = [0] * S
    lens = torch.zeros(S, dtype=torch.int32, device="cuda")
    freq = K.rope_inv_freq(d)
    for step in range(steps):
        live = [step >= f for f in first]
        n = [x + 1 if on else 0 for x, on in zip(n, live)]
        pos = i32(*(step - f if on else -1 for f, on in zip(first, live)))
        lens.copy_(i32(*n))
        for c in caches:
            for s in range(S):
                c.reserve(s, n[s])
        x = randn(S, 512, seed=60 + step)
        mass = [c.mass.clone() for c in caches]
        stack.forward(x, caches=caches, positions=pos, seq_lens=lens, slots=lens - 1)
        for i, c in enumerate(caches[:1]):          # the first layer's input is x
            xn = K.rms_norm(x, stack.attention_norms[i], stack.eps)
            a = stack.attention[i]
            for s in range(S):
                if not live[s]:
                    continue
                q, _ = normed((mats[i][0] @ xn[s].double()).view(1, hq, d), a.q_norm, a.norm_eps, False)
                q, _ = rotate(q, pos[s:s + 1], freq, False)
                t = torch.arange(n[s], device="cuda")
                pages = c.block_table[s][t // page].long()
                kd = c.k[pages, t % page].double() * ks
                z = torch.einsum("hd,nhd->hn", q[0], kd.repeat_interleave(hq // hkv, 1)) * d ** -0.5
                p, tol = weights(q[0], kd, torch.logsumexp(z, -1), d ** -0.5)
                want = mass[i][s, :, :n[s]].double()
                want[:, -1] = 0.0                   # the new token's
                want = want + p
                # q is off by its f32 projection, as in the test of the plain steps
                slack = p * q.abs().sum(-1).max() * kd.abs().max() * d ** -0.5 * 2.0 ** -15
                assert ((c.mass[s, :, :n[s]] - want).abs() <= tol + slack + want * 2.0 ** -23).all()
                held = c.held[s, :, :n[s]]
                assert (held[:, -1] == pos[s]).all()
                assert (held.sort(-1).values.diff(dim=-1) > 0).all()       # each token once
        if step % every == every - 1:
            moves = [evict_plain(n, c.mass.cpu(), c.held.cpu(), keep, recent) for c in caches]
            old = [(c.mass.clone(), c.held.clone(), c.k.clone(), c.v.clone()) for c in caches]
            attention.evict(caches, lens, keep, recent, max_len=40)
            n = [min(x, keep) for x in n]
            assert lens.tolist() == n
            for c, mv, (m, h, k, v) in zip(caches, moves, old):
                for (s, head), (a, b) in mv.items():
                    for x0, x1 in zip(a, b):
                        m[s, head, x1], h[s, head, x1] = m[s, head, x0], h[s, head, x0]
                        p0, p1 = (c.block_table[s, y // page].long() for y in (x0, x1))
                        for cc in (k, v):
                            z = cc.view(torch.uint8) if dtype == E4M3 else cc
                            z[p1, x1 % page, head] = z[p0, x0 % page, head]
                bits = torch.uint8 if dtype == E4M3 else torch.int16
                assert torch.equal(c.mass, m) and torch.equal(c.held, h)
                assert torch.equal(c.k.view(bits), k.view(bits))
                assert torch.equal(c.v.view(bits), v.view(bits))
                for s in range(S):
                    c.trim(s, n[s])
                assert c.free_pages == 40 - sum(-(-x // page) for x in n)
    for c in caches:
        assert c.device_status() == 0
    for a in stack.attention:
        assert a.device_status() == 0


def test_cut_step_captured():
    """A step with its eviction in one graph: one slot is taken and one given up."""
    keep, S = 16, 2
    stack, _ = normed_decoder(F16)
    caches, eager = ([PagedKVCache(12, 4, 2, 64, S, 6, F16, track=True) for _ in range(2)]
                     for _ in range(2))
    for c in caches + eager:
        for s in range(S):
            c.reserve(s, keep + 1)
    out, x = torch.zeros(S, 512, device="cuda"), torch.zeros(S, 512, device="cuda")
    pos, lens = i32(0, 0), i32(0, 0)
    slots = torch.zeros_like(lens)

    def step(cs, lens, slots, out):
        slots.copy_(lens)
        lens.add_(1)
        stack.forward(x, out=out, caches=cs, positions=pos, seq_lens=lens, slots=slots,
                      max_len=keep + 1)
        return attention.evict(cs, lens, keep, 4, max_len=keep + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(eager, lens.clone(), slots.clone(), out)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(caches, lens, slots, out)
    for c, e in zip(caches, eager):                 # the captured calls have not run
        e.k.copy_(c.k), e.v.copy_(c.v), e.mass.copy_(c.mass), e.held.copy_(c.held)
    lens2, slots2, out2 = torch.zeros_like(lens), torch.zeros_like(slots), torch.zeros_like(out)
    for i in range(3 * keep):
        x.copy_(randn(S, 512, seed=i))
        pos.fill_(i)
        g.replay()
        step(eager, lens2, slots2, out2)
        assert torch.equal(out, out2) and lens.tolist() == lens2.tolist() == [min(i + 1, keep)] * S
        for c, e in zip(caches, eager):
            assert torch.equal(c.mass, e.mass) and torch.equal(c.held, e.held)
    assert all(c.device_status() == 0 for c in caches)


def test_prompt_outlives_the_sequence_that_brought_it():
    """Sequences go on behind a prompt's pages, eager and in a captured step, when the prompt's own
    sequence has been released and its place holds another prompt."""
    S, tokens, hkv, d, page = 64, 8192, 2, 64, 64
    width = tokens // page + 1
    stack, _ = normed_decoder(F16)
    caches = [PagedKVCache(2 * width + S, page, hkv, d, S + 1, width, F16) for _ in range(2)]

    def bring(seed):
        for li, c in enumerate(caches):
            c.reserve(S, tokens)
            c.append(None, randn(tokens, hkv, d, seed=seed + li), randn(tokens, hkv, d, seed=seed + 9 + li),
                     torch.arange(tokens, dtype=torch.int32, device="cuda"),
                     seq_ids=torch.full((tokens,), S, dtype=torch.int32, device="cuda"))
    bring(1)
    for c in caches:
        for s in range(S):
            c.share(s, S, tokens)
            c.reserve(s, tokens + 1)
    x, out = randn(S, 512, seed=3), torch.zeros(S, 512, device="cuda")
    pos, lens = i32(*[tokens] * S), i32(*[tokens + 1] * S)
    prefixes = [c.prefix(S, tokens) for c in caches]

    def step(lists):
        return stack.forward(x, out=out, caches=caches, positions=pos, seq_lens=lens, prefixes=lists,
                             max_len=tokens + 1)
    want = step(prefixes).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(prefixes)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step([c.prefix(0, tokens) for c in caches])         # made above: the same lists
    for other in (None, 20):
        for c in caches:
            c.release(S)
        if other:
            bring(other)
        for again in (lambda: step(prefixes), lambda: step([c.prefix(5, tokens) for c in caches]),
                      g.replay):
            out.zero_()
            again()
            assert torch.equal(out, want)
    assert all(c.device_status() == 0 for c in caches)
    assert all(a.device_status() == 0 for a in stack.attention)
    c = caches[0]
    with pytest.raises(RuntimeError, match="before a capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            x.add_(0.0)
            c.prefix(S, 2 * page)


def test_first_step_behind_a_prefix_captured():
    """The workspace of the first call of a size is not one that only the graph's replays clear:
    steps outside of the graph, before it is replayed and after, give the same."""
    S, tokens, page = 33, 4096, 64
    width = tokens // page + 1
    stack, _ = normed_decoder(F16)
    caches = [PagedKVCache(width + S, page, 2, 64, S + 1, width, F16) for _ in range(2)]
    for li, c in enumerate(caches):
        c.reserve(S, tokens)
        c.append(None, randn(tokens, 2, 64, seed=li), randn(tokens, 2, 64, seed=5 + li),
                 torch.arange(tokens, dtype=torch.int32, device="cuda"),
                 seq_ids=torch.full((tokens,), S, dtype=torch.int32, device="cuda"))
        for s in range(S):
            c.share(s, S, tokens)
            c.reserve(s, tokens + 1)
    x, out = randn(S, 512, seed=3), torch.zeros(S, 512, device="cuda")
    pos, lens = i32(*[tokens] * S), i32(*[tokens + 1] * S)
    prefixes = [c.prefix(S, tokens) for c in caches]
    kw = dict(out=out, caches=caches, positions=pos, seq_lens=lens, max_len=tokens + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                   # everything but the prefix
        stack.forward(x, **kw)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        stack.forward(x, prefixes=prefixes, **kw)
    assert not any(a._prefix_ws for a in stack.attention)
    stack.forward(x, prefixes=prefixes, **kw)
    want = out.clone()
    for again in (g.replay, lambda: stack.forward(x, prefixes=prefixes, **kw), g.replay, g.replay):
        out.zero_()
        again()
        assert torch.equal(out, want)
    assert all(a._prefix_ws and a.device_status() == 0 for a in stack.attention)
    assert all(c.device_status() == 0 for c in caches)
    caches[0].block_table[3, width - 1] = -1        # reported by replays too
    g.replay()
    assert caches[0].device_status() == K.STATUS_BAD_PAGE and caches[1].device_status() == 0
