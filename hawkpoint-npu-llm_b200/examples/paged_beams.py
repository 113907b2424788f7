#!/usr/bin/env python3
"""A decoder over the paged K/V cache operators, and beams that share a prompt.

    python hawkpoint-npu-llm_b200/examples/paged_beams.py [--model tiny-qwen] [--prompt 300] [--beams 4] [--new 24]

The prompt is prefilled once, in chunks; ``fork`` starts every beam from its
pages (whole pages shared, the last one copied); the beams decode together, a
token each a step, and after some steps the better half is forked over the
rest; ``free`` and ``compact`` then leave the pool as a long-running program
would want it.  Nothing of the cache's books passes through the host.

Projections run on ``hb_tc_gemm``, norms and SwiGLU are torch element-wise, with
the reference's BF16 rounding points (npu_llm/runtime/cpu_backend.py:131-181);
the model is any object with the package surface of runtime/model.py.
"""

import argparse
import ctypes
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parents[1]
if str(PKG) not in sys.path:
    sys.path.insert(0, str(PKG))

import numpy as np  # noqa: E402
import torch  # noqa: E402

from runtime import hb_lib, layout  # noqa: E402
from runtime.b200_engine import rope_tables  # noqa: E402
from runtime.paged_kv import PAGE, PagedKVCache  # noqa: E402
from runtime.synthetic import shape_from_metadata  # noqa: E402

MAX_ROWS = 256  # rows of one hb_tc_gemm


class Projection:
    """y = W x of BF16 rows on the tensor cores; FP32 out."""

    def __init__(self, matrix, device):
        self.rows, self.k = matrix.shape
        self.weight = torch.from_numpy(layout.pack_matrix_bytes(matrix)).to(device)
        self.lib = hb_lib.load()
        self.scratch = torch.zeros(self.lib.hb_tc_gemm_scratch_bytes(self.rows, self.k, MAX_ROWS), dtype=torch.uint8,
                                   device=device)

    def __call__(self, x):
        y = torch.empty((x.shape[0], self.rows), dtype=torch.float32, device=x.device)
        stream = torch.cuda.current_stream(x.device).cuda_stream
        for at in range(0, x.shape[0], MAX_ROWS):
            part = x[at: at + MAX_ROWS]
            n = part.shape[0]
            packed = torch.zeros(((n + 7) // 8 * 8, self.k), dtype=torch.bfloat16, device=x.device)
            packed[:n] = part
            packed = packed.view(-1, 8, self.k // 8, 8).transpose(1, 2).contiguous()
            hb_lib.check(self.lib.hb_tc_gemm(
                self.weight.data_ptr(), self.rows, self.k, packed.data_ptr(), n,
                ctypes.cast(y[at:].data_ptr(), ctypes.POINTER(ctypes.c_float)), self.scratch.data_ptr(),
                self.scratch.numel(), stream))
        return y


class PagedDecoder:
    """The layers of a model over a ``PagedKVCache``."""

    def __init__(self, model, n_slots, max_context, n_pages, device=None):
        s = self.shape = shape_from_metadata(model.metadata)
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.device = device
        self.cache = PagedKVCache(s.layers, s.kv_heads, s.head_dim, n_pages, n_slots, max_context, device=device)
        fp32 = lambda name: torch.from_numpy(np.asarray(model.raw(name), np.float32)).to(device)  # noqa: E731
        proj = lambda name: Projection(model.bf16_projection(name), device)  # noqa: E731
        self.embedding = fp32("token_embedding").bfloat16()
        self.layers = []
        for i in range(s.layers):
            p = f"layer{i:02d}"
            self.layers.append(dict(
                input_norm=fp32(f"{p}.input_norm"), post_attn_norm=fp32(f"{p}.post_attn_norm"),
                bias=fp32(f"{p}.qkv_bias") if f"{p}.qkv_bias" in model.tensors else None,
                **{name: proj(f"{p}.{name}") for name in ("qkv", "o_proj", "gate_up", "down_proj")}))
        self.final_norm, self.lm_head = fp32("final_norm"), proj("lm_head")
        cos, sin = rope_tables(s.rope_theta, s.head_dim, self.cache.table.shape[1] * PAGE)
        self.cos, self.sin = torch.from_numpy(cos).to(device), torch.from_numpy(sin).to(device)

    def _norm(self, x, gamma):
        v = x.float()
        return (v * (1.0 / torch.sqrt(v.square().mean(1, keepdim=True) + self.shape.rms_eps)) * gamma).bfloat16()

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def step(self, slots, counts, tokens):
        """New rows of several sequences: slot ``slots[b]`` continues with the
        next ``counts[b]`` of ``tokens`` (device tensor of ids).  Returns the
        FP32 logits of each sequence's last row."""
        counts = list(counts)
        starts = np.concatenate([[0], np.cumsum(counts)])
        slots_d, row_start = self.ints(slots), self.ints(starts)
        self.cache.reserve(slots_d, self.ints(counts))
        h = self.embedding[tokens]
        for i, w in enumerate(self.layers):
            qkv = w["qkv"](self._norm(h, w["input_norm"])).bfloat16()
            if w["bias"] is not None:
                qkv = (qkv.float() + w["bias"]).bfloat16()
            q = self.cache.append(i, qkv, slots_d, row_start, max(counts), self.cos, self.sin)
            o = self.cache.attend(i, q, slots_d, row_start, max(counts))
            h1 = (w["o_proj"](o.flatten(1)).bfloat16().float() + h.float()).bfloat16()
            gate, up = w["gate_up"](self._norm(h1, w["post_attn_norm"])).bfloat16().float().chunk(2, 1)
            act = (gate / (1.0 + torch.exp(-gate.clamp(-80.0, 80.0))) * up).bfloat16()
            h = (w["down_proj"](act).bfloat16().float() + h1.float()).bfloat16()
        last = h[row_start[1:].long() - 1]
        return self.lm_head(self._norm(last, self.final_norm))

    def prefill(self, slot, tokens, chunk=256):
        """A prompt in chunks; the last position's logits."""
        for at in range(0, len(tokens), chunk):
            part = tokens[at: at + chunk]
            logits = self.step([slot], [len(part)], part)
        return logits[0]


def beams(decoder, prompt, n_beams, new_tokens, swap_at=8):
    """Beams over one prompt: the n_beams best first tokens, each continued
    greedily; after every ``swap_at`` tokens the better half takes the other
    half's place.  Returns (tokens [n_beams, new_tokens], log-probabilities)."""
    cache = decoder.cache
    first = decoder.prefill(0, prompt)
    scores, token = torch.log_softmax(first.double(), 0).topk(n_beams)
    # every beam starts on the prompt's pages: whole pages shared, the last one its own
    slots = list(range(1, n_beams + 1))
    cache.fork(decoder.ints([0] * n_beams), decoder.ints(slots), decoder.ints([len(prompt)] * n_beams))
    cache.free(decoder.ints([0]))
    out = token[:, None]
    for t in range(1, new_tokens):
        logits = decoder.step(slots, [1] * n_beams, token)
        logp = torch.log_softmax(logits.double(), 1)
        best, token = logp.max(1)
        scores = scores + best
        out = torch.cat([out, token[:, None]], 1)
        if t % swap_at == 0 and n_beams > 1:
            order = scores.argsort(descending=True)
            parent = order[torch.arange(n_beams, device=order.device) % ((n_beams + 1) // 2)]
            lengths = cache.lengths[parent + 1]
            cache.fork((parent + 1).int(), decoder.ints(slots), lengths.contiguous())
            out, scores, token = out[parent], scores[parent], token[parent]
    return out, scores


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--model", default="tiny-qwen")
    parser.add_argument("--prompt", type=int, default=300)
    parser.add_argument("--beams", type=int, default=4)
    parser.add_argument("--new", type=int, default=24)
    args = parser.parse_args(argv)
    from runtime import synthetic

    model = synthetic.build(args.model, seed=1)
    context = args.prompt + args.new
    pages = -(-context // PAGE)
    decoder = PagedDecoder(model, args.beams + 1, context, pages * (args.beams + 1) + 2 * args.beams)
    prompt = torch.tensor(synthetic.prompt_ids(model.shape.vocab, args.prompt, seed=2), device="cuda")
    tokens, scores = beams(decoder, prompt, args.beams, args.new)
    cache = decoder.cache
    held = int((cache.refs > 0).sum())
    moved = int((cache.compact() != torch.arange(cache.refs.numel(), device="cuda")).logical_and(cache.refs > 0).sum())
    cache.status()
    for row, score in zip(tokens.tolist(), scores.tolist()):
        print(f"{score:10.3f}  {row}")
    print(f"{args.beams} beams of {context - 1} positions hold {held} of {args.beams * pages} pages; "
          f"{moved} page indices changed in the compaction")
    cache.free(decoder.ints(list(range(args.beams + 1))))
    cache.status()


if __name__ == "__main__":
    main()
