"""QwenMoeModel: the whole Qwen1.5-MoE decoder on one B200 (runtime/
qwen_moe.py:233-432), its routed experts paged through the HBM expert cache.

Per layer, as the reference's forward: input RMSNorm, attention (int8 q/k/v
with biases, RoPE, a KV cache, causal softmax attention, int8 o), the
residual, post-attention RMSNorm, the MoE block, the residual; then the
final norm and the int8 lm_head. Everything stays on the device: the
residual adds are fused into the next norm (er_rms_norm), RoPE writes the
rotated keys and the values straight into the cache (er_rope_kv), the
embedding rows are dequantized on the device (er_embed_int8), the
projections stream their int8 weights (er_int8_linear), attention is
er_attention, and the MoE block is PagedMoeStack.moe: the router and top-k
on the device, the selected experts made resident in the cache (copies from
pinned host records on the cache's copy stream), the Fate prefetch of the
next layer's guesses when a policy is given, and the block on the cached
records. Only the expert ids cross to the host each layer, to drive the
cache, as in the reference.

With a PagedKVCache in place of a KVCache, the keys and values of many
sequences lie in pages (fp32 or bf16): one call may carry tokens of several
sequences, or trees of drafted tokens, and attention runs over the pages
(expertrelay_b200.kv). On it stand generate_drafted (several tokens a call,
where a draft has guessed them) and beam_search.
"""

from __future__ import annotations

import time
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib, beam, draft as drafts
from .cache import HbmExpertCache, HostRecords
from .kv_cache import PagedKVCache
from .paged import PagedMoeStack
from .prefetch import PrefetchPolicy
from .trace import PHASE_DECODE, PHASE_PREFILL


@dataclass(frozen=True)
class ModelConfig:
    """The config.json fields the forward pass uses (runtime/qwen_moe.py:53-87)."""

    vocab_size: int
    hidden_size: int
    num_layers: int
    num_heads: int
    num_kv_heads: int
    num_experts: int
    top_k: int
    norm_topk_prob: bool
    rms_norm_eps: float
    rope_theta: float
    moe_intermediate_size: int
    shared_expert_intermediate_size: int

    @property
    def head_dim(self) -> int:
        return self.hidden_size // self.num_heads

    @classmethod
    def from_hf(cls, c: dict) -> ModelConfig:
        if c.get("use_sliding_window"):
            raise NotImplementedError("sliding-window attention is not implemented")
        if c.get("mlp_only_layers") or c.get("decoder_sparse_step", 1) != 1:
            raise NotImplementedError("dense (non-MoE) decoder layers are not implemented")
        return cls(c["vocab_size"], c["hidden_size"], c["num_hidden_layers"], c["num_attention_heads"],
                   c["num_key_value_heads"], c["num_experts"], c["num_experts_per_tok"], bool(c["norm_topk_prob"]),
                   float(c["rms_norm_eps"]), float(c["rope_theta"]), c["moe_intermediate_size"],
                   c["shared_expert_intermediate_size"])


class KVCache:
    """Keys and values of every layer on the device: [layers, max_seq,
    kv_heads, head_dim] fp32 each (runtime/qwen_moe.py:90-106)."""

    def __init__(self, config: ModelConfig, max_seq: int, device):
        shape = (config.num_layers, max_seq, config.num_kv_heads, config.head_dim)
        self.k = torch.zeros(shape, dtype=torch.float32, device=device)
        self.v = torch.zeros(shape, dtype=torch.float32, device=device)
        self.length = 0
        self.max_seq = max_seq

    @property
    def nbytes(self) -> int:
        return 2 * self.k.numel() * 4


def _dev(a, dtype, device) -> torch.Tensor:
    return torch.as_tensor(np.ascontiguousarray(a)).to(device=device, dtype=dtype)


class QwenMoeModel:
    """host: an expertrelay_b200.synth.HostModel (or anything with its
    fields); records: the routed experts as [layers, experts, record_size]
    uint8 (pinned host memory; default: the host blocks' records);
    cache_records: HBM slots for routed records (default: all of them);
    prefetch: the Fate policy's prefetch of the next layer's experts;
    prefetch_adaptive: cap the prefetch's copies on one-token calls at what
    fits in each layer's measured window (runtime/generate.py:112)."""

    def __init__(self, host, *, records: torch.Tensor | None = None, cache_records: int | None = None,
                 prefetch: bool = False, prefetch_adaptive: bool = False, device="cuda",
                 path: int = _lib.PATH_AUTO):
        if not torch.cuda.is_available():
            raise RuntimeError("QwenMoeModel needs a CUDA device (the B200 path has no CPU fallback)")
        self.device = dev = torch.device(device)
        if dev.index is None:
            self.device = dev = torch.device("cuda", torch.cuda.current_device())
        self.c = c = ModelConfig.from_hf(host.config)
        self.path = path
        self.embed_q, self.embed_s = _dev(host.embed[0], torch.int8, dev), _dev(host.embed[1], torch.float32, dev)
        self.head_q, self.head_s = _dev(host.lm_head[0], torch.int8, dev), _dev(host.lm_head[1], torch.float32, dev)
        self.final_norm = _dev(host.final_norm, torch.float32, dev)
        self.layers = []
        for lay in host.layers:
            w = {"in_norm": _dev(lay.input_norm, torch.float32, dev), "post_norm": _dev(lay.post_norm, torch.float32, dev)}
            # q, k and v as one projection (rows stacked: one weight stream, one launch)
            qkv = ("q_proj", "k_proj", "v_proj")
            w["qkv"] = (_dev(np.concatenate([lay.proj[m][0] for m in qkv]), torch.int8, dev),
                        _dev(np.concatenate([lay.proj[m][1] for m in qkv]), torch.float32, dev))
            w["qkv_bias"] = _dev(np.concatenate([lay.bias[m] for m in qkv]), torch.float32, dev)
            w["o_proj"] = (_dev(lay.proj["o_proj"][0], torch.int8, dev), _dev(lay.proj["o_proj"][1], torch.float32, dev))
            self.layers.append(w)
        if records is None:
            records = HostRecords.from_blocks(host.blocks)
        else:
            records = HostRecords(records, host.blocks[0].layout, pin=True)
        self.records = records
        rs = records.layout.record_size
        slots = cache_records if cache_records is not None else records.layers * records.experts
        self.cache = HbmExpertCache(records, capacity_bytes=slots * rs, device=dev)
        policy = PrefetchPolicy(top_k=c.top_k) if prefetch else None
        self.stack = PagedMoeStack(host.blocks, self.cache, prefetcher=policy, norm_topk_prob=c.norm_topk_prob)
        self.stack.prefetch_adaptive = prefetch_adaptive
        self._bad = torch.zeros(1, dtype=torch.int32, device=dev)

    def close(self) -> None:
        self.cache.close()

    def new_cache(self, max_seq: int) -> KVCache:
        return KVCache(self.c, max_seq, self.device)

    def new_paged_cache(self, seqs: int, max_seq: int, **options) -> PagedKVCache:
        """A cache for `seqs` sequences of up to max_seq places each (PagedKVCache's options)."""
        return PagedKVCache(self.c, seqs, max_seq, device=self.device, **options)

    def _stream(self) -> int:
        return torch.cuda.current_stream(self.device).cuda_stream

    def _linear(self, x: torch.Tensor, qs, bias: torch.Tensor | None = None) -> torch.Tensor:
        q, s = qs
        n, out_dim, in_dim = x.shape[0], q.shape[0], q.shape[1]
        y = torch.empty((n, out_dim), dtype=torch.float32, device=self.device)
        _lib.check(_lib.lib().er_int8_linear(x.data_ptr(), in_dim, q.data_ptr(), s.data_ptr(),
                                             None if bias is None else bias.data_ptr(), y.data_ptr(), n, out_dim,
                                             in_dim, self._stream()), "er_int8_linear")
        return y

    def _norm(self, x: torch.Tensor, w: torch.Tensor, add: torch.Tensor | None = None) -> torch.Tensor:
        """h = rms_norm(x (+ add)); with `add`, x itself becomes x + add."""
        n, H = x.shape
        h = torch.empty_like(x)
        _lib.check(_lib.lib().er_rms_norm(x.data_ptr(), None if add is None else add.data_ptr(), w.data_ptr(),
                                          self.c.rms_norm_eps, n, H, x.data_ptr(), h.data_ptr(), self._stream()),
                   "er_rms_norm")
        return h

    def _attention(self, layer: int, h: torch.Tensor, kv, allowed) -> torch.Tensor:
        """allowed: the causal mask of a KVCache, or the Step of a PagedKVCache."""
        c, w = self.c, self.layers[layer]
        n, d = h.shape[0], c.head_dim
        qkv = self._linear(h, w["qkv"], w["qkv_bias"])
        if isinstance(kv, PagedKVCache):
            out = kv.attend(layer, allowed, qkv, c.num_heads, c.rope_theta)
            return self._linear(out.view(n, c.num_heads * d), w["o_proj"])
        q = torch.empty((n, c.num_heads * d), dtype=torch.float32, device=self.device)
        start, end = kv.length, kv.length + n
        _lib.check(_lib.lib().er_rope_kv(qkv.data_ptr(), qkv.shape[1], q.data_ptr(), n, c.num_heads, c.num_kv_heads,
                                         d, start, c.rope_theta, kv.k[layer].data_ptr(), kv.v[layer].data_ptr(),
                                         kv.max_seq, self._stream()), "er_rope_kv")
        keys, values = kv.k[layer, :end], kv.v[layer, :end]
        if c.num_kv_heads != c.num_heads:
            rep = c.num_heads // c.num_kv_heads
            keys, values = keys.repeat_interleave(rep, dim=1), values.repeat_interleave(rep, dim=1)
        out = torch.empty((n, c.num_heads * d), dtype=torch.float32, device=self.device)
        _lib.check(_lib.lib().er_attention(q.data_ptr(), keys.contiguous().data_ptr(), values.contiguous().data_ptr(),
                                           allowed.data_ptr(), out.data_ptr(), n, end, c.num_heads, d,
                                           self._stream()), "er_attention")
        return self._linear(out, w["o_proj"])

    def forward(self, token_ids, kv: KVCache | PagedKVCache, *, all_logits: bool = False, expert_trace=None,
                seqs=None, parents=None) -> torch.Tensor:
        """Run `token_ids` after what `kv` holds; logits [vocab] of the last
        position (or [n, vocab] with all_logits), on the device. With a
        PagedKVCache, `seqs` names the sequence of every token (default: all
        of sequence 0), and a call that raises leaves it as it was. `parents`
        makes the tokens trees of drafted ones (PagedKVCache.step): each sees
        its sequence, its ancestors and itself; kv.drafted is then the step
        that kv.accept needs."""
        c = self.c
        ids = torch.as_tensor(np.asarray(token_ids, dtype=np.int64)).to(self.device)
        n = ids.shape[0]
        if isinstance(kv, PagedKVCache):
            seqs = np.zeros(n, dtype=np.int64) if seqs is None else np.asarray(seqs, dtype=np.int64)
            if seqs.shape != (n,):
                raise ValueError(f"seqs: one sequence for each of {n} tokens, got {seqs.shape}")
            if expert_trace is not None and len(np.unique(seqs)) > 1:
                raise ValueError("a trace follows one sequence")
            if expert_trace is not None and parents is not None:
                raise ValueError("a trace follows one text: not with parents")
            step = kv.step(seqs, parents)
            try:
                return self._forward(token_ids, ids, kv, step, int(kv.pages.position[seqs[0]]) - n, all_logits,
                                     expert_trace)
            except BaseException:  # the places of a call that fails hold nothing, or not in every layer
                kv.undo(step)
                raise
        if seqs is not None or parents is not None:
            raise ValueError("seqs, parents: only with a PagedKVCache")
        if kv.length + n > kv.max_seq:
            raise ValueError(f"sequence length {kv.length + n} exceeds the KV cache ({kv.max_seq})")
        # causal: query start + i sees keys 0 .. start + i (the same for every layer)
        start, end = kv.length, kv.length + n
        allowed = (torch.arange(end, device=self.device)[None, :]
                   <= (start + torch.arange(n, device=self.device))[:, None]).to(torch.uint8)
        return self._forward(token_ids, ids, kv, allowed, start, all_logits, expert_trace)

    def _forward(self, token_ids, ids, kv, allowed, start: int, all_logits: bool, expert_trace) -> torch.Tensor:
        """forward() from position `start` on; allowed as for _attention."""
        c, n = self.c, ids.shape[0]
        x = torch.empty((n, c.hidden_size), dtype=torch.float32, device=self.device)
        _lib.check(_lib.lib().er_embed_int8(self.embed_q.data_ptr(), self.embed_s.data_ptr(), c.vocab_size,
                                            c.hidden_size, ids.data_ptr(), n, x.data_ptr(), self._bad.data_ptr(),
                                            self._stream()), "er_embed_int8")
        if expert_trace is not None:
            positions = start + np.arange(n)
            expert_trace.begin(positions, np.asarray(token_ids), PHASE_PREFILL if start == 0 else PHASE_DECODE)
        h = self._norm(x, self.layers[0]["in_norm"])
        for layer in range(c.num_layers):
            a = self._attention(layer, h, kv, allowed)
            h = self._norm(x, self.layers[layer]["post_norm"], add=a)
            y = self.stack.moe(layer, h, self.path, trace=expert_trace)
            if layer + 1 < c.num_layers:
                h = self._norm(x, self.layers[layer + 1]["in_norm"], add=y)
        if not isinstance(kv, PagedKVCache):
            kv.length += n
        if expert_trace is not None:
            expert_trace.end()
        rows = slice(None) if all_logits else slice(n - 1, n)
        xf, yf = x[rows].contiguous(), y[rows].contiguous()
        final = self._norm(xf, self.final_norm, add=yf)
        logits = self._linear(final, (self.head_q, self.head_s))
        if int(self._bad.item()):
            self._bad.zero_()
            raise ValueError(f"token ids outside [0, {c.vocab_size})")
        return logits if all_logits else logits[0]

    def generate(self, prompt, new_tokens: int, *, max_seq: int | None = None, expert_trace=None, kv=None):
        """Greedy decoding (runtime/generate.py): the prompt in one call, then
        one token per call. Returns (generated ids, seconds of the prompt call,
        seconds per decode call). kv: a cache of one's own (a PagedKVCache's
        sequence 0); otherwise a new KVCache of max_seq positions."""
        prompt = [int(t) for t in prompt]
        if kv is None:
            kv = self.new_cache(max_seq or len(prompt) + new_tokens)
        torch.cuda.synchronize(self.device)
        t0 = time.perf_counter()
        logits = self.forward(prompt, kv, expert_trace=expert_trace)
        tok = int(torch.argmax(logits).item())
        t_prompt = time.perf_counter() - t0
        out, step = [tok], []
        for _ in range(new_tokens - 1):
            t1 = time.perf_counter()
            logits = self.forward([tok], kv, expert_trace=expert_trace)
            tok = int(torch.argmax(logits).item())
            step.append(time.perf_counter() - t1)
            out.append(tok)
        return out, t_prompt, step

    def generate_drafted(self, prompt, new_tokens: int, draft=drafts.from_text, *, kv: PagedKVCache | None = None,
                         seq: int = 0):
        """Greedy decoding, several tokens a call where `draft` has guessed them:
        draft(text) gets the prompt and what has come so far and returns (tokens,
        parents), a tree of guesses at what comes next (kv.attend_tree's order; -1:
        the text's last token; none is fine). One call runs them all, and the
        path that greedy decoding would have taken stays (by that call's logits: they
        are rounded otherwise than those of a call of one token, and drafted tokens
        see all pages of a cache with `select`). Returns (generated ids,
        calls after the prompt's). kv: a cache of one's own, without accumulated
        weights; the prompt goes on from what its sequence `seq` holds (room for
        the prompt, new_tokens and a call's guesses)."""
        prompt = [int(t) for t in prompt]
        if new_tokens < 1:
            raise ValueError(f"new_tokens: at least 1, got {new_tokens}")
        if kv is None:
            kv, seq = self.new_paged_cache(1, len(prompt) + new_tokens + 256), 0
        if kv.mass is not None:
            raise ValueError("generate_drafted: not over a cache made with mass=True, which takes no drafted tokens")
        out, calls = [int(torch.argmax(self.forward(prompt, kv, seqs=[seq] * len(prompt))).item())], 0
        while len(out) < new_tokens:
            tokens, parents = draft(prompt + out)
            # the last token, its guesses behind it; no more than the cache takes, a child never before its parent
            most = min(256, max(1, kv.room(seq)))
            tokens = [out[-1], *map(int, tokens)][:most]
            parents = [-1, *(int(p) + 1 for p in parents)][:most]
            logits = self.forward(tokens, kv, all_logits=True, seqs=[seq] * len(tokens), parents=parents)
            next_of = torch.argmax(logits, dim=1).tolist()
            try:
                kv.check()
            except BaseException:  # the logits are no good
                kv.undo(kv.drafted)
                raise
            path, had = [0], len(out)
            while len(out) < new_tokens:
                out.append(next_of[path[-1]])
                child = next((i for i in range(path[-1] + 1, len(tokens))
                              if parents[i] == path[-1] and tokens[i] == out[-1]), None)
                if child is None:
                    break
                path.append(child)
            kv.accept(kv.drafted, [path[:len(out) - had]])  # like generate's, the cache ends before the last token
            calls += 1
        return out, calls

    def beam_search(self, prompt, beams: int, new_tokens: int, *, end: int | None = None,
                    kv: PagedKVCache | None = None) -> list[tuple[list[int], float]]:
        """The `beams` best continuations of `prompt` by the sum of their tokens' log
        probabilities that a search of that breadth finds, best first: [(ids, sum)].
        They have new_tokens tokens, or end with `end`. kv: a cache of one's own;
        the prompt goes on from what sequence 0 holds, and sequences 1 .. beams - 1
        are empty, for the search's use. What sequences 0 .. beams - 1 hold afterwards
        are beams of its last step: release them."""
        prompt = [int(t) for t in prompt]
        if beams < 1 or new_tokens < 1:
            raise ValueError(f"{beams} beams of {new_tokens} tokens: at least one each")
        if kv is None:
            kv = self.new_paged_cache(beams, len(prompt) + new_tokens)
        kv.pages.known([beams - 1])
        full = [s for s in range(1, beams) if kv.length(s)]
        if full:
            raise ValueError(f"beam_search: sequences {full} of the cache are not empty")
        count = beams if end is None else 2 * beams  # as many that go on, whichever of them end
        if count > 128:
            raise ValueError(f"{beams} beams: at most {128 * beams // count}")
        logits = self.forward(prompt, kv)[None]
        scores, texts, done, live = torch.zeros((1, 1), device=self.device), [[]], [], [0]
        for n in range(new_tokens):
            best, of, tokens = (x[0].tolist() for x in beam.select(logits, scores, min(count, logits.numel())))
            kv.check()
            going = []
            for value, i, t in zip(best, of, tokens):
                if t == end or n + 1 == new_tokens:
                    done.append((texts[i] + [t], value))
                elif len(going) < beams:
                    going.append((value, i, t))
            done = sorted(done, key=lambda d: -d[1])[:beams]
            # sums only fall: nothing that goes on can pass what has ended
            if not going or len(done) == beams and done[-1][1] >= going[0][0]:
                break
            kv.reorder(list(range(len(going))), [live[i] for _, i, _ in going])
            live = list(range(len(going)))
            texts = [texts[i] + [t] for _, i, t in going]
            scores = torch.tensor([[value for value, _, _ in going]], device=self.device)
            logits = self.forward([t for _, _, t in going], kv, all_logits=True, seqs=live)
        return done
