"""KV-cached greedy decoder: replaces the O(L^2) full-recompute loop of VAEShell.greedy_decode
(reference transvae/trans_models.py:383-436) with one memory expansion + 125 single-token steps.

Per step and decoder layer: LayerNorm -> one fused QKV GEMM (M = molecules) -> append K,V to the
cache -> one-query attention over the cache -> output projection (+residual) -> LayerNorm ->
query projection -> one-query attention over the PRE-PROJECTED memory keys/values -> projection
-> LayerNorm -> FFN.  The arg-max is taken on the device; token ids never visit the host.
The arithmetic per position is the same as the reference's (causal masking makes position i
independent of later positions), which is what makes the token sequences bit-identical.

kv_cache="fp8" keeps both caches as e4m3 codes with a scale per (page of 32 tokens, head) (kv8.KV8Cache): a quarter of the
bytes, which is what a step of a large batch is bound by.  Keys and values are then rounded to 3 mantissa bits, so tokens may
differ from the fp32 cache's where the two best logits are close; and a molecule whose source mask is empty gets zeros
from its memory, where the fp32 path attends uniformly as the reference does.
scores=True also returns the log probability of every token and the entropy it was chosen from (loss.token_logprobs).
"""
import collections
import math

import torch

from . import ops
from .kv8 import KV8Cache
from .ops import _p, _stream, call


GRAPH_MAX_N = 2048      # latent batches up to this size are launch-bound: their step loop is replayed as a HIP graph
GRAPH_CACHE_MAX = 4     # captured graphs kept per model (least recently used goes first): a graph owns its K/V caches,
#                         ~1.5 MB per latent for trans4x-256, so an unbounded cache grows by GBs with every new batch size


def clear_decode_graphs(model):
    "drop every captured decode graph of `model` (and the HBM their private pools hold)"
    model.__dict__.pop("_tvae_decode_graphs", None)


def _weights_stamp(model):
    "changes whenever a weight may have changed (in-place updates bump _version; .data writes bump the epoch)"
    return (ops._weights_epoch[0], sum(p._version for p in model.parameters()), ops.compute_dtype())


KV_CACHES = ("fp32", "fp8")


def _cache8(n, tokens, h, dk, device, page=32):
    "an 8-bit cache for `tokens` tokens of n sequences; its memory is not cleared: nothing is read before it is written"
    per = -(-tokens // page)
    k, v = (torch.empty((n * per, h, page, dk), dtype=torch.uint8, device=device) for _ in range(2))
    ke, ve = (torch.empty((n * per, h), dtype=torch.uint8, device=device) for _ in range(2))
    return KV8Cache(k, v, ke, ve, n_seq=n)


class GreedyDecoder:
    def __init__(self, model, h, kv_cache="fp32", scores=False):
        if kv_cache not in KV_CACHES:
            raise ops._lib.TvaeError("kv_cache must be one of %s (got %r)" % (KV_CACHES, kv_cache))
        self.model, self.h, self.kv_cache, self.scores = model, h, kv_cache, bool(scores)

    @staticmethod
    def _ln(x, norm):
        return ops.layernorm_fwd(x, norm.a_2, norm.b_2, norm.eps)

    @torch.no_grad()
    def run(self, z, key_mask, start_id, cond_ids=(), max_len=125):
        """z (n, d_latent) on the device; key_mask (n, 127) uint8 source mask; returns (n, max_len) int64, with scores
        (ids, logp, entropy), the latter two (n, max_len) fp32.

        Small batches (n <= GRAPH_MAX_N) spend their time in ~5000 launches of tiny kernels, so from the second
        call with the same shape on the projections + 125 steps are captured once into a HIP graph (static
        buffers for the memory, the mask and the ids) and replayed; the arithmetic and the kernels are the same."""
        model = self.model
        n = z.shape[0]
        spec = ops.MaskSpec(key_mask=key_mask)
        mem = model.decoder.expand_memory(z, spec)            # (n, 127, d), already through decoder.norm
        cond_ids = tuple(int(t) for t in cond_ids)
        if n > GRAPH_MAX_N or not torch.cuda.is_available():
            return self._result(self._steps(mem, key_mask, None, start_id, cond_ids, max_len))
        key = (n, tuple(mem.shape), cond_ids, int(start_id), max_len, z.device.index, self.kv_cache, self.scores)
        cache = model.__dict__.setdefault("_tvae_decode_graphs", {"graphs": collections.OrderedDict(), "seen": {}})
        graphs, seen = cache["graphs"], cache["seen"]
        stamp = _weights_stamp(model)
        entry = graphs.get(key)
        if entry is not None and entry["stamp"] != stamp:
            del graphs[key]                                   # weights moved since the capture: take it again
            entry = None
        if entry is None:
            if seen.get(key) != stamp:                        # first call with this shape: plain launches
                if len(seen) > 64:
                    seen.clear()
                seen[key] = stamp
                return self._result(self._steps(mem, key_mask, None, start_id, cond_ids, max_len))
            while len(graphs) >= GRAPH_CACHE_MAX:
                graphs.popitem(last=False)                    # least recently used graph and its pool
            entry = {"stamp": stamp, "mem": torch.empty_like(mem), "mask": torch.empty_like(key_mask),
                     "out": self._buffers(n, max_len, z.device)}
            entry["mem"].copy_(mem)
            entry["mask"].copy_(key_mask)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                self._steps(entry["mem"], entry["mask"], entry["out"], start_id, cond_ids, max_len)
            entry["graph"] = graph
            graphs[key] = entry
        graphs.move_to_end(key)
        entry["mem"].copy_(mem)
        entry["mask"].copy_(key_mask)
        entry["graph"].replay()
        return self._result(entry["out"], clone=True)

    def _buffers(self, n, max_len, device):
        "(ids, logp, entropy) that the steps write; the latter two None without scores"
        ids = torch.empty((n, max_len + 1), dtype=torch.int64, device=device)
        if not self.scores:
            return ids, None, None
        return (ids,) + tuple(torch.empty((n, max_len), dtype=torch.float32, device=device) for _ in range(2))

    def _result(self, out, clone=False):
        ids, logp, ent = out
        ids = ids[:, 1:]
        if clone:
            ids, logp, ent = (None if t is None else t.clone() for t in (ids, logp, ent))
        return (ids, logp, ent) if self.scores else ids

    def _steps(self, mem, key_mask, out, start_id, cond_ids, max_len):
        "source K/V projections + max_len single-token steps; every launch goes to the current stream"
        for out in self._steps_iter(mem, key_mask, out, start_id, cond_ids, max_len):
            pass
        return out

    def run_iter(self, z, key_mask, start_id, cond_ids=(), max_len=125):
        """run() for a large slab as a generator: yields after the set-up and after every token step, the last value is the
        (n, max_len) ids (with scores what run() returns).  VAEShell.decode_latents resumes several of these in turn, each under its own stream, so that one
        piece's attention over its K/V caches (HBM-bound) runs beside another's projections (MFMA-bound).  The caller must
        make the generator's stream current around every next()."""
        spec = ops.MaskSpec(key_mask=key_mask)
        mem = self.model.decoder.expand_memory(z, spec)
        out = None
        for out in self._steps_iter(mem, key_mask, None, start_id, tuple(int(t) for t in cond_ids), max_len):
            yield None
        yield self._result(out)

    def _steps_iter(self, mem, key_mask, out, start_id, cond_ids, max_len):
        "_steps as a generator (yields its buffers after the set-up and after every step)"
        model, h = self.model, self.h
        dec = model.decoder
        dev = mem.device
        n, Ls, d = mem.shape
        dk = d // h
        scale = 1.0 / math.sqrt(dk)
        mem2 = mem.reshape(n * Ls, d)
        T = max_len + 1
        layers = list(dec.layers)
        # source-attention keys/values never change during decoding: project them once
        fp8 = self.kv_cache == "fp8"
        kc, vc, wqkv, bqkv = [], [], [], []
        for lyr in layers:
            lin = lyr.src_attn.linears
            k = ops.linear_fwd(mem2, lin[1].weight, lin[1].bias)
            v = ops.linear_fwd(mem2, lin[2].weight, lin[2].bias)
            if fp8:
                k, v = self._store8(_cache8(n, Ls, h, dk, dev), k, v), None
            kc.append(k)
            vc.append(v)
            sl = lyr.self_attn.linears
            wqkv.append(torch.cat([sl[0].weight, sl[1].weight, sl[2].weight], 0).contiguous())
            bqkv.append(torch.cat([sl[0].bias, sl[1].bias, sl[2].bias], 0).contiguous())
        if fp8:
            ks, vs = [_cache8(n, T, h, dk, dev) for _ in layers], None
        else:
            ks = [torch.empty((n, T, d), device=dev, dtype=torch.float32) for _ in layers]
            vs = [torch.empty((n, T, d), device=dev, dtype=torch.float32) for _ in layers]
        if out is None:
            out = self._buffers(n, max_len, dev)
        ids, logp, ent = out
        ids.fill_(int(start_id))
        for j, t in enumerate(cond_ids):
            ids[:, j + 1] = int(t)
        emb, pos = model.tgt_embed[0], model.tgt_embed[1]
        lut, pe = emb.lut.weight, pos.pe[0]
        vocab = lut.shape[0]
        gen = model.generator.proj
        n_cls = gen.weight.shape[0]
        x = torch.empty((n, d), device=dev, dtype=torch.float32)
        qkv = torch.empty((n, 3 * d), device=dev, dtype=torch.float32)
        att = torch.empty((n, d), device=dev, dtype=torch.float32)
        qkv5, att4 = qkv.view(n, 1, 3, h, dk), att.view(n, 1, h, dk)
        yield out
        for t in range(max_len):
            st = _stream()               # a generator may be resumed under another stream context than it was started in
            call("tvae_embed_step", _p(ids), T, t, _p(lut), _p(pe), _p(x), n, d, vocab, st)
            cur = x
            for li, lyr in enumerate(layers):
                sub = lyr.sublayer
                n0 = self._ln(cur, sub[0].norm)
                ops.linear_fwd(n0, wqkv[li], bqkv[li], out=qkv)
                if fp8:
                    ks[li].store(qkv5[:, :, 1], qkv5[:, :, 2], start=t)
                    ks[li].attend(qkv5[:, :, 0], t + 1, out=att4)
                else:
                    call("tvae_scatter_rows", _p(qkv[:, d:]), 3 * d, _p(ks[li]), d, T, t, n, d, st)
                    call("tvae_scatter_rows", _p(qkv[:, 2 * d:]), 3 * d, _p(vs[li]), d, T, t, n, d, st)
                    call("tvae_decode_attn", _p(qkv), 3 * d, _p(ks[li]), _p(vs[li]), d, T, _p(att), d, None, 0,
                         t + 1, n, h, dk, scale, st)
                so = lyr.self_attn.linears[3]
                cur = ops.linear_fwd(att, so.weight, so.bias, residual=cur)
                n1 = self._ln(cur, sub[1].norm)
                cl = lyr.src_attn.linears
                q = ops.linear_fwd(n1, cl[0].weight, cl[0].bias)
                if fp8:
                    kc[li].attend(q.view(n, 1, h, dk), Ls, key_mask=key_mask, out=att4)
                else:
                    call("tvae_decode_attn", _p(q), d, _p(kc[li]), _p(vc[li]), d, Ls, _p(att), d, _p(key_mask), Ls,
                         Ls, n, h, dk, scale, st)
                cur = ops.linear_fwd(att, cl[3].weight, cl[3].bias, residual=cur)
                n2 = self._ln(cur, sub[2].norm)
                ff = lyr.feed_forward
                hmid = ops.linear_fwd(n2, ff.w_1.weight, ff.w_1.bias, relu=True)
                cur = ops.linear_fwd(hmid, ff.w_2.weight, ff.w_2.bias, residual=cur)
            if t >= len(cond_ids) or self.scores:
                y = self._ln(cur, dec.norm)
                logits = ops.linear_fwd(y, gen.weight, gen.bias)
                if t >= len(cond_ids):
                    call("tvae_argmax_next", _p(logits), n_cls, n_cls, _p(ids), T, t + 1, n, st)
                if self.scores:                              # of the given tokens too; token id 1 is class 0
                    ops.token_logp(logits, ids[:, t + 1], tok_sub=1, out=(logp[:, t], ent[:, t]))
            yield out

    @torch.no_grad()
    def cache_error(self, z, key_mask):
        """(layers, 2): what 8 bits do to the memory's keys and values of the latents z, as |rounded - exact| / |exact| (2-norms over
        the tokens of key_mask), layer by layer.  Stores them as run() would and reads them back."""
        mem = self.model.decoder.expand_memory(z, ops.MaskSpec(key_mask=key_mask))
        n, Ls, d = mem.shape
        seen = (key_mask != 0)[:, :, None, None]
        out = []
        for lyr in self.model.decoder.layers:
            exact = [ops.linear_fwd(mem.reshape(n * Ls, d), lin.weight, lin.bias) for lin in lyr.src_attn.linears[1:3]]
            cache = self._store8(_cache8(n, Ls, self.h, d // self.h, mem.device), *exact)
            for got, x in zip(cache.load(Ls), exact):
                x = x.view(got.shape) * seen
                size = torch.linalg.vector_norm(x)
                out.append(torch.where(size == 0, size, torch.linalg.vector_norm(got * seen - x) / size))    # no token: no error
        return torch.stack(out).view(-1, 2)

    @staticmethod
    def _store8(cache, k, v):
        "k, v (n * tokens, h * dk), projections of every token, into an empty cache"
        n = cache.n_seq
        cache.store(k.view(n, -1, cache.heads, cache.dk), v.view(n, -1, cache.heads, cache.dk))
        return cache
