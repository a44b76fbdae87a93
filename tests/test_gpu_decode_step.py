"""One decoder layer and the output head through the package's operators, as a server runs them: norm ->
Q/K/V pack -> rotary + KV append -> attention -> output projection -> add + norm -> MoE FFN -> norm -> head
-> sampling.  A shared prefix is prefilled once, prompts of uneven lengths behind it in one call, then
tokens are decoded from one captured graph whose lengths advance in place.

Every stage of the new operators is checked against float64 on the GPU's own inputs to it (so that no
tolerance compounds), and every replay against an eager step from the same state."""

import numpy as np
import pytest

from gpu_helpers import build_pair, log
from kv_helpers import HALF_STEP, norm_reference, rotate_reference, sample_reference
from pgmoe.synth import CONFIGS, random_blocks

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

H, HQ, HKV, D, V, PS, PREFIX = 1024, 8, 2, 128, 4096, 16, 37
Q4_K, Q6_K = 12, 14


class Layer:
    def __init__(self, dev):
        from pgmoe import FusedLinearPack, GGUFQuantLinear, GGUFRMSNorm, HipPagedKVCache, HipRotary

        rng = np.random.default_rng(3)

        def lin(qt, n, k, mode):
            return GGUFQuantLinear(mode, k, n, qt, raw=random_blocks(rng, qt, n, k, 0.02), device=dev)

        self.pack = FusedLinearPack([lin(Q4_K, HQ * D, H, "w4"), lin(Q4_K, HKV * D, H, "w4"), lin(Q4_K, HKV * D, H, "w4")])
        self.o = lin(Q4_K, H, HQ * D, "w4")
        self.head = lin(Q6_K, V, H, "w8")
        self.embed = (torch.from_numpy(rng.standard_normal((V, H)).astype(np.float32))).to(dev)
        self.norms = [GGUFRMSNorm(torch.from_numpy(1 + 0.1 * rng.standard_normal(H).astype(np.float32)).to(dev))
                      for _ in range(3)]
        self.qn, self.kn = (torch.from_numpy(1 + 0.2 * rng.standard_normal(D).astype(np.float32)).to(dev) for _ in range(2))
        self.moe = build_pair(CONFIGS["tiny"], seed=0, scale=0.01)[2]
        self.rope = HipRotary(D, base=1e6, device=dev)
        self.cache = HipPagedKVCache(64, PS, HKV, D, device=dev)

    def step(self, tokens, batch, keep=None):
        """Logits of the given tokens [T]; keep: a dict that receives the inner tensors."""
        x = self.embed[tokens]
        parts = self.pack(self.norms[0](x, out_dtype=torch.float16))
        q, k, v = (p.unflatten(1, (-1, D)) for p in parts)
        qr = self.cache.append(q, k, v, batch, self.rope, q_norm=self.qn, k_norm=self.kn)
        a = self.cache.attend(qr, batch)
        h, n = self.norms[1].forward_with_residual(x, self.o(a.flatten(1)).float())
        h, n = self.norms[2].forward_with_residual(h, self.moe(n[None])[0])
        logits = self.head(n).float()
        if keep is not None:
            keep.update(q=q, k=k, v=v, qr=qr, a=a, logits=logits)
        return logits


def _check_stage(lay, got, seqs, new):
    """append and attend of one call: seqs [(table row, own keys, tokens in this call)] in order."""
    pos, rows = [], []
    for table, own, n in seqs:
        for i in range(n):
            j = own - n + i
            pos.append(new["prefix"] + j)
            rows.append((int(table[j // PS]), j % PS))
    inv = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    pg, ro = (torch.tensor(x) for x in zip(*rows))
    k, v = lay.cache.k.cpu(), lay.cache.v.cpu()
    for y, x, w in ((got["qr"].cpu(), got["q"], lay.qn), (k[pg, :, ro], got["k"], lay.kn)):
        ref, mag = rotate_reference(norm_reference(x[:len(pos)].cpu(), w.cpu()), torch.tensor(pos), inv, False)
        assert bool(((y[:len(pos)].double() - ref).abs() <= HALF_STEP[torch.float16] * ref.abs() + 32 * 2.0 ** -24 * mag + 2.0 ** -25).all())
    assert torch.equal(v[pg, :, ro], got["v"][:len(pos)].cpu().half())
    t, G = 0, HQ // HKV
    pre = [(int(new["pages"][j // PS]), j % PS) for j in range(new["prefix"])]
    for table, own, n in seqs:
        for i in range(n):
            at = pre + [(int(table[j // PS]), j % PS) for j in range(own - n + i + 1)]
            p, r = (torch.tensor(x) for x in zip(*at))
            for h in range(HKV):
                q = got["qr"][t, h * G:(h + 1) * G].cpu().double()
                kk, vv = k[p, h, r].double(), v[p, h, r].double()
                x = q @ kk.T / D ** 0.5
                w = torch.softmax(x, -1)
                o = w @ vv
                ds = 2.0 ** -24 * ((D + 4) * (q.abs() @ kk.abs().T).amax() / D ** 0.5 + 3 * x.abs().amax())
                tol = HALF_STEP[torch.float16] * o.abs() + (w @ vv.abs()) * (1.01 * HALF_STEP[torch.float16] + 2 * ds +
                                                                             2 * (len(at) + 64) * 2.0 ** -24) + 2.0 ** -25
                assert bool(((got["a"][t, h * G:(h + 1) * G].cpu().double() - o).abs() <= tol).all()), (t, h)
            t += 1


def test_prefill_and_captured_decode():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from pgmoe import KVBatch, sample_tokens

    dev = torch.device("cuda", 0)
    log("decode step: prefill")
    lay = Layer(dev)
    g = torch.Generator().manual_seed(0)
    order = torch.randperm(64, generator=g, dtype=torch.int32)
    shared, tables = order[:3].tolist(), order[3:3 + 4 * 5].view(4, 5)
    # the prefix itself: one sequence whose own keys it is
    toks = torch.randint(0, V, (PREFIX,), generator=g).to(dev)
    got = {}
    lay.step(toks, KVBatch([shared], [PREFIX], q_start=[0, PREFIX], device=dev), got)
    _check_stage(lay, got, [(shared, PREFIX, PREFIX)], dict(prefix=0, pages=[]))
    # four prompts behind it in one call, two rows of padding at the end
    lens = [11, 1, 30, 16]
    start = [0, 11, 12, 42, 58]
    toks = torch.randint(0, V, (60,), generator=g).to(dev)
    dlens = torch.tensor(lens, dtype=torch.int32, device=dev)
    dtab = tables.to(dev)
    pages = torch.tensor(shared, dtype=torch.int32, device=dev)
    got = {}
    logits = lay.step(toks, KVBatch(dtab, dlens, q_start=start, prefix_pages=pages, prefix_len=PREFIX), got)
    _check_stage(lay, got, [(tables[b], lens[b], lens[b]) for b in range(4)], dict(prefix=PREFIX, pages=shared))

    # decode: lengths advance in the graph, the sampled tokens are the next step's input
    batch = KVBatch(dtab, dlens, prefix_pages=pages, prefix_len=PREFIX)
    u = torch.zeros(4, device=dev)
    last = torch.tensor([s - 1 for s in start[1:]], device=dev)
    par = dict(temperature=0.7, top_k=50, top_p=0.95, min_p=0.01)
    u.copy_(torch.rand(4, generator=g))
    cur, _ = sample_tokens(logits[last].contiguous(), u, **par)
    inner = {}

    def decode():
        batch.lens.add_(1)
        x = lay.step(cur, batch, inner)
        tok, lp = sample_tokens(x, u, **par)
        inner.update(tok=tok, lp=lp)
        cur.copy_(tok)

    state = (batch.lens, cur, lay.cache.k, lay.cache.v)
    before = [t.clone() for t in state]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        decode()  # the stream's workspaces exist before capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            decode()
    captured = dict(inner)
    torch.cuda.synchronize()
    for t, b in zip(state, before):
        t.copy_(b)
    for rep in range(8):
        log(f"decode step: replay {rep}")
        u.copy_(torch.rand(4, generator=g))
        torch.cuda.synchronize()
        before = [t.clone() for t in state]
        decode()  # eager, then the graph from the same state
        torch.cuda.synchronize()
        want = {n: t.clone() for n, t in inner.items()}
        after = [t.clone() for t in state]
        for t, b in zip(state, before):
            t.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for n, t in want.items():
            assert torch.equal(t, captured[n]), (rep, n)
        for t, a in zip(state, after):
            assert torch.equal(t, a), rep
        lens = [n + 1 for n in lens]
        assert batch.lens.tolist() == lens
        _check_stage(lay, captured, [(tables[b], lens[b], 1) for b in range(4)], dict(prefix=PREFIX, pages=shared))
        for b in range(4):
            t, p = sample_reference(captured["logits"][b].cpu().double().numpy(), float(u[b]), *par.values())
            assert int(captured["tok"][b]) == t
            assert abs(float(captured["lp"][b]) - p) <= 2.0 ** -23 * abs(p) + 2.0 ** -38
    del graph
