"""Several conversations of one model over a paged KV cache.

    python examples/paged_sessions.py

Runs a small Qwen3-shaped model (random weights in raw ggml blocks) with the
package's kernels: the projections through matmul_batch, every layer's
attention through the paged-cache operators.  A shared opening is prefilled
once; each conversation names its pages in its own block table and continues
in pages of its own; then all of them decode together, one token a step, with
the step captured in a CUDA graph.  The logits are compared with a Session's,
whose cache is fp32 and contiguous.
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import rpgbarengine_b200 as rb  # noqa: E402
from rpgbarengine_b200 import synth  # noqa: E402


class PagedQwen3:
    """The shape's layers over one PagedKV per layer (16-bit pages)."""

    def __init__(self, shape, tensors, n_pages: int, page_size: int, dtype=torch.bfloat16, ops=rb):
        self.shape, self.dtype, self.ops = shape, dtype, ops
        self.w = {t.name: (t.ggml_type, torch.from_numpy(np.ascontiguousarray(t.data).view(np.uint8)).cuda(), t.dims) for t in tensors}
        self.caches = [rb.PagedKV.empty(n_pages, page_size, shape.n_kv_heads, shape.head_dim, dtype) for _ in range(shape.n_layers)]
        self.rope = rb.rope_table(shape.context_length, shape.head_dim, shape.rope_theta)
        ty, data, _ = self.w["token_embd.weight"]
        self.embd = rb.dequantize_rows(ty, data, shape.vocab, shape.hidden)

    def gain(self, name):
        return self.w[name][1].view(torch.float32)

    def matmul(self, name, x):
        ty, data, dims = self.w[name]
        return rb.matmul_batch(ty, data, int(dims[1]), int(dims[0]), x)

    def norm(self, x, name):
        return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.shape.rms_eps) * self.gain(name)).contiguous()

    def forward(self, ids, batch):
        """Hidden states of the batch's packed rows `ids`, whose K and V go into the pages."""
        s, decode = self.shape, batch.keep[2] is None
        attend = self.ops.paged_attention_decode if decode else self.ops.paged_attention_prompt
        x = self.embd[ids]
        n = x.shape[0]
        for l, cache in enumerate(self.caches):
            p = f"blk.{l}."
            h = self.norm(x, p + "attn_norm.weight")
            q = self.matmul(p + "attn_q.weight", h).view(n, s.n_heads, s.head_dim)
            k = self.matmul(p + "attn_k.weight", h).view(n, s.n_kv_heads, s.head_dim)
            v = self.matmul(p + "attn_v.weight", h).view(n, s.n_kv_heads, s.head_dim)
            q = self.ops.paged_append(cache, batch, q, k, v, self.gain(p + "attn_q_norm.weight"),
                                      self.gain(p + "attn_k_norm.weight"), s.rms_eps, self.rope)
            a = attend(cache, batch, q)
            x = x + self.matmul(p + "attn_output.weight", a.float().view(n, -1))
            h = self.norm(x, p + "ffn_norm.weight")
            g = torch.nn.functional.silu(self.matmul(p + "ffn_gate.weight", h)) * self.matmul(p + "ffn_up.weight", h)
            x = x + self.matmul(p + "ffn_down.weight", g.contiguous())
        return x

    def logits(self, x):
        name = "output.weight" if "output.weight" in self.w else "token_embd.weight"
        return self.matmul(name, self.norm(x, "output_norm.weight"))


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def run(shape=synth.TINY_MIX, seed=5, page=16, opening=40, own=(17, 1, 33), steps=12, dtype=torch.float16, ops=rb):
    """Returns (paged logits of each step, tokens, the prompts) of the conversations."""
    tensors = synth.build_tensors(shape, seed)
    prefix = synth.prompt_ids(seed, opening, shape.vocab)
    tails = [synth.prompt_ids(seed + 1 + i, n, shape.vocab) for i, n in enumerate(own)]
    n = len(own)
    shared = opening // page  # whole pages of the opening, held once by all conversations
    per = -(-(opening + max(own) + steps) // page)
    net = PagedQwen3(shape, tensors, 1 + -(-opening // page) + n * per, page, dtype, ops)
    with torch.inference_mode():
        # the opening, a whole prompt of its own, into pages 1, 2, ..
        opening_pages = [1 + i for i in range(-(-opening // page))]
        batch = rb.PagedBatch(i32([opening_pages]), i32([opening]), i32([0, opening]), opening)
        net.forward(torch.as_tensor(np.asarray(prefix), device="cuda").long(), batch)
        # each conversation: the shared pages, then its own; what the opening left in
        # its last, unfilled page is prefilled again into a page of the conversation
        free = iter(range(1 + len(opening_pages), 10 ** 6))
        table = i32([opening_pages[:shared] + [next(free) for _ in range(per - shared)] for _ in range(n)])
        new = [np.concatenate([prefix[shared * page:], t]) for t in tails]
        cu = np.concatenate([[0], np.cumsum([len(t) for t in new])]).astype(np.int32)
        lens = i32([opening + len(t) for t in tails])
        batch = rb.PagedBatch(table, lens, torch.from_numpy(cu).cuda(), int(cu[-1]))
        ids = torch.as_tensor(np.concatenate(new), device="cuda").long()
        x = net.forward(ids, batch)
        out = [net.logits(x[torch.from_numpy(cu[1:] - 1).long().cuda()])]
        # decode: every conversation one token a step, one captured graph for all steps
        token = out[0].argmax(-1)
        tokens = [token.tolist()]
        step = rb.PagedBatch(table, lens)

        def one():
            lens.add_(1)
            return net.logits(net.forward(token, step))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # once outside the graph: workspaces and kernels are set up
            one()
            lens.sub_(1)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = one()
        for _ in range(steps - 1):
            graph.replay()
            out.append(logits.clone())
            token.copy_(out[-1].argmax(-1))
            tokens.append(token.tolist())
    prompts = [np.concatenate([prefix, t]).astype(np.int32) for t in tails]
    return torch.stack(out), tokens, prompts, tensors


def compare(shape, logits, tokens, prompts, tensors):
    """Relative L2 error of every conversation's logits against a Session's fed the same tokens."""
    model = rb.Model.upload(shape, tensors, 0, shape.context_length)
    worst = 0.0
    for i, p in enumerate(prompts):
        s = model.session(len(p) + len(tokens))
        want = [s.forward_full(p)]
        for t in tokens[:-1]:
            want.append(s.forward_full([t[i]]))
        got = logits[:, i].double().cpu().numpy()
        w = np.asarray(want, np.float64)
        worst = max(worst, float((np.linalg.norm(got - w, axis=1) / np.linalg.norm(w, axis=1)).max()))
    return worst


def main():
    shape = synth.TINY_MIX
    for dtype in (torch.float16, torch.bfloat16):
        logits, tokens, prompts, tensors = run(shape, dtype=dtype)
        err = compare(shape, logits, tokens, prompts, tensors)
        print(f"{str(dtype)[6:]} pages: {len(prompts)} conversations, {len(tokens)} tokens each, "
              f"logits within {err:.2e} (relative L2) of fp32 sessions")
        for i, p in enumerate(prompts):
            print(f"  conversation {i}: {len(p)} prompt tokens, then {[t[i] for t in tokens]}")


if __name__ == "__main__":
    main()
