"""Plain, slow decoding over an 8-bit cache with eviction, one sequence at a time: the layers of `mistral_plain`, the cache as its
definition says (levels and scales of finished blocks, the unfinished one as it came, weights from the one-token steps, eviction per
layer and head), CPU float32.  It shares no code with the package under test."""
from __future__ import annotations

import torch

from plain import mistral_plain as P

BLOCK = 16


def quantized(x, fmt):
    """What a block x [16, D] stands for once it is held in 8 bits."""
    top = 127.0 if fmt == "int8" else 448.0
    scale = max(float(x.abs().max()) / top, 2.0 ** -126)
    q = torch.clamp(x / scale, -top, top)
    return (torch.round(q) if fmt == "int8" else q.to(torch.float8_e4m3fn).float()) * scale


class BlockDecoder:
    def __init__(self, cfg, w, fmt, rnd=P.no_rounding):
        self.cfg, self.w, self.fmt, self.rnd = cfg, w, fmt, rnd
        L, G = cfg["num_hidden_layers"], cfg["num_key_value_heads"]
        # per layer and head: finished blocks [k, v, weight]; rows of the unfinished block (k, v); the weight it has so far
        self.blocks = [[[] for _ in range(G)] for _ in range(L)]
        self.tail = [[[] for _ in range(G)] for _ in range(L)]
        self.tail_weight = [[0.0] * G for _ in range(L)]
        self.pos, self.steps = 0, 0

    @property
    def held(self):
        return BLOCK * len(self.blocks[0][0]) + len(self.tail[0][0])

    def _append(self, layer, h, k, v):
        self.tail[layer][h].append((k, v))

    def _finish(self, layer, h):
        t = self.tail[layer][h]
        if len(t) == BLOCK:
            k, v = (torch.stack([r[i] for r in t]) for i in range(2))
            self.blocks[layer][h].append([quantized(k, self.fmt), quantized(v, self.fmt), self.tail_weight[layer][h]])
            self.tail[layer][h], self.tail_weight[layer][h] = [], 0.0

    def _layer_weights(self, layer):
        p = f"model.layers.{layer}."
        return p, {n: self.w[p + f"self_attn.{n}_proj.weight"] for n in "qkvo"}

    def prompt(self, ids):
        """Logits of the last row; the prompt attends over its keys and values as they come."""
        cfg, rnd = self.cfg, self.rnd
        x = P.embed(self.w["model.embed_tokens.weight"], ids, 1.0)
        for layer in range(cfg["num_hidden_layers"]):
            p, a = self._layer_weights(layer)
            xn = rnd(P.rmsnorm(x, self.w[p + "input_layernorm.weight"], cfg["rms_norm_eps"]))
            y, parts = P.attention_layer(xn, a["q"], a["k"], a["v"], a["o"], heads=cfg["num_attention_heads"], kv_heads=cfg["num_key_value_heads"],
                                         head_dim=cfg["head_dim"], rope_theta=cfg["rope_theta"], window=cfg.get("sliding_window"), rnd=rnd,
                                         return_parts=True)
            for t in range(len(ids)):
                for h in range(cfg["num_key_value_heads"]):
                    self._append(layer, h, parts["k"][t, h], parts["v"][t, h])
                    self._finish(layer, h)
            x = self._rest(x + y, p)
        self.pos = len(ids)
        return self._head(x[-1:])

    def step(self, token):
        """Logits after one more token."""
        cfg, rnd = self.cfg, self.rnd
        H, G, D = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"]
        x = P.embed(self.w["model.embed_tokens.weight"], [token], 1.0)
        for layer in range(cfg["num_hidden_layers"]):
            p, a = self._layer_weights(layer)
            xn = rnd(P.rmsnorm(x, self.w[p + "input_layernorm.weight"], cfg["rms_norm_eps"]))
            q, k, v = (rnd(P.matmul(xn, a[n])).view(1, -1, D) for n in "qkv")
            q, k = (rnd(P.rope_sequence(t, cfg["rope_theta"], D, D, "half", first_pos=self.pos)) for t in (q, k))
            out = torch.zeros(H, D)
            for g in range(G):
                self._append(layer, g, k[0, g], v[0, g])
                blocks, tail = self.blocks[layer][g], self.tail[layer][g]
                ks, vs = (torch.cat([b[i] for b in blocks] + [torch.stack([r[i] for r in tail])]) for i in range(2))
                n = ks.shape[0]
                first = max(0, n - cfg["sliding_window"]) if cfg.get("sliding_window") else 0
                for h in range(g * H // G, (g + 1) * H // G):
                    s = (q[0, h] @ ks[first:].t()) * D ** -0.5
                    pr = torch.zeros(n)
                    pr[first:] = P.softmax(s)
                    out[h] = pr @ vs
                    for b, block in enumerate(blocks):
                        block[2] += float(pr[b * BLOCK:(b + 1) * BLOCK].sum())
                    self.tail_weight[layer][g] += float(pr[len(blocks) * BLOCK:].sum())
                self._finish(layer, g)
            x = self._rest(x + P.matmul(rnd(out.reshape(1, H * D)), a["o"]), p)
        self.pos += 1
        self.steps += 1
        return self._head(x)

    def evict(self, keep, recent, every):
        """The policy, after a step; True if the sequence went back."""
        if self.steps < every or self.held < keep + every:
            return False
        for layer in self.blocks:
            for g, blocks in enumerate(layer):
                n, r = len(blocks), recent // BLOCK
                order = sorted(range(n - r), key=lambda b: (-blocks[b][2], b))[:keep // BLOCK - r]
                layer[g] = [blocks[b] for b in sorted(order) + list(range(n - r, n))]
        self.steps = 0
        return True

    def _rest(self, x, p):
        cfg, w = self.cfg, self.w
        xn = self.rnd(P.rmsnorm(x, w[p + "post_attention_layernorm.weight"], cfg["rms_norm_eps"]))
        return x + P.ffn_layer(xn, w[p + "mlp.gate_proj.weight"], w[p + "mlp.up_proj.weight"], w[p + "mlp.down_proj.weight"], self.rnd)

    def _head(self, x):
        hn = self.rnd(P.rmsnorm(x, self.w["model.norm.weight"], self.cfg["rms_norm_eps"]))
        head = self.w["model.embed_tokens.weight"] if self.cfg.get("tie_word_embeddings") else self.w["lm_head.weight"]
        return P.matmul(hn, head)[0]
