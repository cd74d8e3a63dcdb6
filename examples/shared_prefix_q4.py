"""Several answers from one prompt over a 4-bit KV cache with shared pages.

A small seeded Llama-shaped decoder with per-head query/key norms, built from the library's kernel
entry points: the prompt is written once, forked into several sequences that share its pages, every
answer is decoded in one batch, finished answers give their pages back and the pool is compacted.

    python examples/shared_prefix_q4.py [--prompt 200] [--answers 6] [--tokens 24]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vulkan-symbiote-loader_b200"))
import vsl  # noqa: E402

CONFIG = dict(n_layers=4, d_model=512, n_heads=8, n_kv=2, head_dim=64, ffn=1376, vocab=4096, rope_theta=10000.0,
              eps=1e-5)
CHUNK = 16  # prompt rows, or sequences of a step, per pass (vsl_gemv takes up to 16)


class Decoder:
    """Weights, paged 4-bit cache and page bookkeeping of up to n_seq sequences."""

    def __init__(self, cfg=CONFIG, n_seq=8, max_seq=512, n_pages=64, page=64, seed=0):
        self.cfg, self.n_seq, self.page, self.n_pages = cfg, n_seq, page, n_pages
        self.max_pages = -(-max_seq // page)
        c, dev = cfg, dict(device="cuda")
        d, hd, nh, nkv = c["d_model"], c["head_dim"], c["n_heads"], c["n_kv"]
        self.width = (nh + 2 * nkv) * hd

        def weight(tid, rows, cols):
            w = torch.empty(rows, cols, dtype=torch.float16, **dev)
            vsl.synth_fill(w, vsl.F16, seed, tid, 0, rows * cols, 1.0 / math.sqrt(cols))
            return w

        gen = torch.Generator(device="cuda").manual_seed(seed)
        ones = torch.ones(d, **dev)
        self.norm, self.embed, self.head = ones, weight(1, c["vocab"], d), weight(2, c["vocab"], d)
        self.layers = []
        for i in range(c["n_layers"]):
            t = 16 * (i + 1)
            self.layers.append(dict(qkv=weight(t, self.width, d), o=weight(t + 1, d, nh * hd),
                                    gu=weight(t + 2, 2 * c["ffn"], d), down=weight(t + 3, d, c["ffn"]),
                                    q_norm=0.5 + torch.rand(hd, generator=gen, **dev),
                                    k_norm=0.5 + torch.rand(hd, generator=gen, **dev)))
        page_bytes = vsl.kv_page_bytes(vsl.Q4_0, nkv, hd, page)
        self.pools = torch.zeros(2 * c["n_layers"], n_pages, page_bytes, dtype=torch.uint8, **dev)
        self.table = torch.full((n_seq, self.max_pages), -1, dtype=torch.int32, **dev)
        self.lens = torch.zeros(n_seq, dtype=torch.int32, **dev)
        self.ref = torch.zeros(n_pages, dtype=torch.int32, **dev)
        self.status = torch.zeros(1, dtype=torch.int32, **dev)
        self.kv = vsl.KvPages(self.table, n_seq, self.max_pages, page, self.ref, n_pages, list(self.pools), page_bytes,
                              lens=self.lens)
        self.page_ws = torch.zeros(vsl.kv_pages_workspace_size(n_seq, n_pages), dtype=torch.uint8, **dev)
        ws = max(vsl.flash_decode_q4_workspace_size(1, CHUNK, nh, nkv, hd),
                 vsl.flash_decode_q4_workspace_size(min(n_seq, CHUNK), 1, nh, nkv, hd))
        self.attn_ws = torch.zeros(ws, dtype=torch.uint8, **dev)
        ang = torch.arange(max_seq, dtype=torch.float64, **dev)[:, None] * c["rope_theta"] ** (
            -torch.arange(0, hd, 2, dtype=torch.float64, **dev) / hd)
        self.cos, self.sin = ang.cos().float(), ang.sin().float()

    def _ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def extend(self, seqs, add):
        """Pages for `add` more positions of every sequence in seqs; their lengths go up."""
        vsl.kv_extend(self.kv, self._ints(seqs), self._ints([add] * len(seqs)), len(seqs), self.page_ws,
                      self.page_ws.numel(), status=self.status, stream=self._stream())

    def fork(self, src, targets):
        vsl.kv_fork(self.kv, self._ints([src] * len(targets)), self._ints(targets), len(targets), self.page_ws,
                    self.page_ws.numel(), status=self.status, stream=self._stream())

    def free(self, seqs):
        vsl.kv_free(self.kv, self._ints(seqs), len(seqs), status=self.status, stream=self._stream())

    def compact(self):
        """Moves the pages in use to the pool's start; returns (in use, moved)."""
        counts = self._ints([0, 0])
        vsl.kv_compact(self.kv, self.table, self.ref, counts, self.page_ws, self.page_ws.numel(), status=self.status,
                       stream=self._stream())
        return tuple(counts.tolist())

    def pages_in_use(self):
        return int((self.ref > 0).sum())

    @staticmethod
    def _stream():
        return torch.cuda.current_stream().cuda_stream

    def forward(self, ids, seq, pos, batch, rows):
        """Logits of batch x rows tokens (ids int32 on the GPU, sequence by sequence) at positions pos of
        sequences seq; sequence i of the batch has table row seq[i * rows]."""
        c, st, n = self.cfg, self._stream(), batch * rows
        d, hd, nh, nkv = c["d_model"], c["head_dim"], c["n_heads"], c["n_kv"]
        x, qkv, q, attn, act = (torch.empty(n, w, device="cuda") for w in (d, self.width, nh * hd, nh * hd, c["ffn"]))
        table, first = self.table[seq[::rows].long()], pos[::rows].contiguous()
        vsl.embed_gather(vsl.F16, self.embed, c["vocab"], d, ids, n, x, stream=st)
        for i, w in enumerate(self.layers):
            k_cache, v_cache = self.pools[2 * i], self.pools[2 * i + 1]
            vsl.gemv(vsl.F16, w["qkv"], self.width, d, x, n, qkv, vsl.EPI_STORE, self.norm, c["eps"], stream=st)
            vsl.qk_norm_rope_append(qkv, self.width, n, nh, nkv, hd, w["q_norm"], w["k_norm"], c["eps"], seq, pos,
                                    self.n_seq, self.cos, self.sin, self.cos.shape[0], vsl.ROPE_ADJACENT, q, k_cache,
                                    v_cache, vsl.Q4_0, self.n_pages, self.table, self.max_pages, self.page,
                                    status=self.status, stream=st)
            vsl.flash_decode_q4(q, k_cache, v_cache, self.n_pages, table, self.max_pages, self.page, first, batch, rows,
                                nh, nkv, hd, attn, self.attn_ws, self.attn_ws.numel(), status=self.status, stream=st)
            vsl.gemv(vsl.F16, w["o"], d, nh * hd, attn, n, x, vsl.EPI_ADD, stream=st)
            vsl.gemv(vsl.F16, w["gu"], 2 * c["ffn"], d, x, n, act, vsl.EPI_SWIGLU, self.norm, c["eps"], stream=st)
            vsl.gemv(vsl.F16, w["down"], d, c["ffn"], act, n, x, vsl.EPI_ADD, stream=st)
        logits = torch.empty(n, c["vocab"], device="cuda")
        vsl.gemv(vsl.F16, self.head, c["vocab"], d, x, n, logits, vsl.EPI_STORE, self.norm, c["eps"], stream=st)
        return logits

    def prompt(self, ids, seq):
        """Writes a prompt into an empty sequence; logits of its last token."""
        self.extend([seq], len(ids))
        for at in range(0, len(ids), CHUNK):
            part = ids[at:at + CHUNK]
            n = len(part)
            logits = self.forward(self._ints(part), torch.full((n,), seq, dtype=torch.int32, device="cuda"),
                                  torch.arange(at, at + n, dtype=torch.int32, device="cuda"), 1, n)
        return logits[-1]

    def step(self, ids, seqs):
        """One token for each sequence in seqs (one at least); their logits."""
        self.extend(seqs, 1)
        logits = []
        for at in range(0, len(seqs), CHUNK):
            seq = self._ints(seqs[at:at + CHUNK])
            logits.append(self.forward(self._ints(ids[at:at + CHUNK]), seq, (self.lens[seq.long()] - 1).contiguous(),
                                       len(seq), 1))
        return torch.cat(logits)

    def check(self):
        """Raises what the kernels reported: a pool that ran out of pages, positions past the cache."""
        if self.status.item():
            raise RuntimeError("device status %d" % self.status.item())


def answers(dec, prompt, n, tokens, share=True):
    """n answers of `tokens` ids: the k-th starts with the k-th best first token and goes on greedily.
    share=False writes the prompt into every sequence instead of forking it."""
    logits = dec.prompt(prompt, 0)
    first = logits.topk(n).indices.tolist()
    if share:
        dec.fork(0, list(range(1, n)))
    else:
        for s in range(1, n):
            dec.prompt(prompt, s)
    out, all_logits = [first], []
    for _ in range(tokens - 1):
        lg = dec.step(out[-1], list(range(n)))
        all_logits.append(lg)
        out.append(lg.argmax(-1).tolist())
    return [list(a) for a in zip(*out)], all_logits


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--answers", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=24)
    a = ap.parse_args(argv)
    if min(a.prompt, a.answers, a.tokens) < 1 or a.answers > CONFIG["vocab"]:
        ap.error("--prompt, --answers and --tokens are at least 1, --answers at most %d" % CONFIG["vocab"])
    page = 64  # pages: the prompt's once, and for every answer its last one and those of its tokens
    dec = Decoder(n_seq=a.answers, max_seq=a.prompt + a.tokens, page=page,
                  n_pages=-(-a.prompt // page) + a.answers * (2 + a.tokens // page))
    prompt = [(i * 2654435761 >> 7) % CONFIG["vocab"] for i in range(a.prompt)]
    got, _ = answers(dec, prompt, a.answers, a.tokens)
    dec.check()
    for i, ids in enumerate(got):
        print("answer %d: %s" % (i, ids))
    unshared = a.answers * -(-(a.prompt + a.tokens - 1) // dec.page)
    print("pages in use: %d shared, %d unshared" % (dec.pages_in_use(), unshared))
    dec.free(list(range(0, a.answers, 2)))
    print("after freeing every other answer: %d in use, %d moved" % dec.compact())
    if a.answers > 1:
        lg = dec.step([ids[-1] for ids in got[1::2]], list(range(1, a.answers, 2)))
        dec.check()
        print("next tokens of the others: %s" % lg.argmax(-1).tolist())


if __name__ == "__main__":
    main()
