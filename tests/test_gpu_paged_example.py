"""The paged-cache operators together, as examples/paged_sessions.py uses them:
every call against its definition on the inputs that it gets there, and the
logits against sessions with an fp32 cache.

What a 16-bit cache costs the logits depends on the model: q and k are rounded
before scores as large as sqrt(head_dim) are formed, and random K-quant weights
amplify that from layer to layer until two roundings of the same values give
logits that are further from each other than from the session's.  So the
sessions are compared on the 8-bit shape, which does not, and the bound is
measured beside the result: the same conversations with the same 16-bit pages,
but with every operator in elementary torch operations.  The kernels may be
three times as far from the sessions as that (both errors are a few hundred
roundings that fall differently), and no further."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from rpgbarengine_b200 import synth  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Plain:
    """The operators from their definitions, over the same pages."""

    @staticmethod
    def rows(batch):
        table, lens, cu, _ = batch.keep
        n = torch.arange(batch.n_tokens, device="cuda")
        if cu is None:
            return table, n, (lens - 1).long()
        seq = torch.searchsorted(cu.long(), n, right=True) - 1
        return table, seq, (lens.long()[seq] - cu.long()[seq + 1] + n)

    @staticmethod
    def paged_append(cache, batch, q, k, v, q_norm, k_norm, eps, rope):
        table, seq, pos = Plain.rows(batch)

        def turned(x, g):
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * g
            c, s = rope[pos, None].chunk(2, -1)
            a, b = x.chunk(2, -1)
            return torch.cat([a * c - b * s, b * c + a * s], -1).to(cache.dtype)

        page, slot = table[seq, pos // cache.page_size].long(), pos % cache.page_size
        cache.k[page, slot], cache.v[page, slot] = turned(k, k_norm), v.to(cache.dtype)
        return turned(q, q_norm)

    @staticmethod
    def attention(cache, batch, q):
        table, seq, pos = Plain.rows(batch)
        k, v = (x[table.long()].flatten(1, 2)[seq].double().nan_to_num(0, 0, 0) for x in (cache.k, cache.v))  # [row, place, head, dim]
        G = q.shape[1] // k.shape[2]
        s = torch.einsum("nhgd,nthd->nhgt", q.double().view(q.shape[0], -1, G, q.shape[2]), k) * q.shape[2] ** -0.5
        s = s.masked_fill(torch.arange(k.shape[1], device="cuda") > pos[:, None, None, None], float("-inf"))
        return torch.einsum("nhgt,nthd->nhgd", s.softmax(-1), v).reshape(q.shape).to(cache.dtype)

    paged_attention_prompt = paged_attention_decode = attention


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected without a CUDA device")
    spec = importlib.util.spec_from_file_location("paged_sessions", os.path.join(ROOT, "examples", "paged_sessions.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def errors(example, shape, **kw):
    """(kernels, elementary operations): relative L2 of the logits against fp32 sessions."""
    logits, tokens, prompts, tensors = example.run(shape, **kw)
    assert torch.isfinite(logits).all()
    got = example.compare(shape, logits, tokens, prompts, tensors)
    want = example.compare(shape, *example.run(shape, ops=Plain, **kw))
    print(f"{shape.name}: kernels {got:.2e}, elementary operations {want:.2e}")
    return got, want


class Both:
    """Every operator beside its plain form on the same inputs: the kernel's result goes on, the largest
    error over its bound is kept.  Bounds: append rounds once (u of the value, and fp32 arithmetic within
    2^-20 of the row's largest); attention rounds its output and its probabilities (u each of the largest
    visible |v|, which bounds sum p |v|), a quarter of that for the fp32 in between."""

    def __init__(self, dtype):
        import rpgbarengine_b200 as rb
        self.rb, self.u, self.over = rb, {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype], []

    def paged_append(self, cache, batch, q, k, v, *a):
        got = self.rb.paged_append(cache, batch, q, k, v, *a)
        table, seq, pos = Plain.rows(batch)
        page, slot = table[seq, pos // cache.page_size].long(), pos % cache.page_size
        have = [got, cache.k[page, slot].clone(), cache.v[page, slot].clone()]
        want = [Plain.paged_append(cache, batch, q, k, v, *a), cache.k[page, slot], cache.v[page, slot]]
        for g, w in zip(have, want):  # (both are rounded: one unit apart at most where the fp32 values straddle)
            w = w.double()
            self.over.append(((g.double() - w).abs() / (2 * self.u * w.abs() + 2.0 ** -19 * w.abs().amax(-1, keepdim=True))).nan_to_num(0).max())
        cache.k[page, slot], cache.v[page, slot] = have[1], have[2]
        return got

    def attention(self, call, cache, batch, q):
        got, want = call(cache, batch, q), Plain.attention(cache, batch, q).double()
        table, seq, pos = Plain.rows(batch)
        v = cache.v[table.long()].flatten(1, 2)[seq].double()
        far = torch.arange(v.shape[1], device="cuda") > pos[:, None]
        top = v.masked_fill(far[:, :, None, None], 0).abs().amax((1, 2, 3))[:, None, None]
        self.over.append(((got.double() - want).abs() / (1.25 * self.u * (2 * want.abs() + top))).max())
        return got

    def paged_attention_prompt(self, *a):
        return self.attention(self.rb.paged_attention_prompt, *a)

    def paged_attention_decode(self, *a):
        return self.attention(self.rb.paged_attention_decode, *a)


CASES = [dict(shape=synth.TINY_MIX), dict(shape=synth.TINY_UNTIED), dict(shape=synth.TINY_Q8),
         # nothing of the opening fills a page: every conversation prefills it itself
         dict(shape=synth.TINY_MIX, page=64, opening=20, own=(5, 70), steps=5)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_every_call_agrees_with_its_plain_form(example, case, dtype):
    both = Both(dtype)
    example.run(dtype=dtype, ops=both, **CASES[case])
    assert len(both.over) > 20
    assert float(torch.stack(both.over).max()) <= 1


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_paged_conversations_match_sessions(example, dtype):
    got, want = errors(example, synth.TINY_Q8, dtype=dtype)
    assert got <= 3 * want, (got, want)
