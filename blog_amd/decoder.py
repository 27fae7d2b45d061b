"""A Qwen2-architecture decoder over the quantized-linear path: the harness of benchmark configuration C3.

Qwen2.5-0.5B architecture (24 layers, hidden 896, 14 query / 2 KV heads of 64, SwiGLU FFN 4864,
vocabulary 151936, RMSNorm eps 1e-6, rotary theta 1e6), every linear in Q8_0, random-init weights
N(0, 0.02) before quantization (ggml's Q8_0 rule: d = amax / 127 stored as f16, q = round(x / d), ties
away from zero).  The embedding table is tied to the output head and quantized like the linears, so
the lookup dequantizes one Q8_0 row (qlin_launch_quant_embedding) and the head is a Q8_0 GEMV.  No
q/k/v biases.  Norm weights are bf16 values 1 + N(0, 0.1).

Every linear, the embedding lookup and the argmax are qlin.h entry points; RMSNorm, rotary embedding
with the KV-cache store and attention are qlin_decoder.h's.  The prompt runs as one batched pass (the
m > 1 matmuls); each decode step is one token at a position held in device memory, so a step can be
captured into a HIP graph and replayed, the argmax writing the next step's token id on the device.
torch provides the device memory and the streams.

Two variations of the architecture: ``qk_norm`` norms every query and key head before the rotation (weights ``q_norm``
and ``k_norm`` [head_dim] in each layer), and ``kv8`` keeps keys and values in the 8-bit cache of blocks.  With
``set_controls`` the pick goes by the logits after penalties for repeated tokens, biases and a mask; with ``set_adapters``
low-rank adapters stand beside the linears; ``step_drafts`` checks drafted tokens against the model's probabilities in one pass.
"""
from __future__ import annotations

from dataclasses import dataclass

from . import qlin

Q8_0 = 8
QK8_0 = 32


@dataclass
class Qwen2Config:
    layers: int = 24
    hidden: int = 896
    n_heads: int = 14
    kv_heads: int = 2
    head_dim: int = 64
    ffn: int = 4864
    vocab: int = 151936
    eps: float = 1e-6
    theta: float = 1e6
    wtype: int = Q8_0
    qk_norm: bool = False  # norms of query and key heads
    kv8: bool = False      # the cache in 8 bits (head_dim 64, 96, 128, 192 or 256)

    @property
    def q_dim(self) -> int:
        return self.n_heads * self.head_dim

    @property
    def kv_dim(self) -> int:
        return self.kv_heads * self.head_dim


def quantize_q8_0(torch, x):
    """ggml's Q8_0 quantizer (quantize_row_q8_0_ref) of a [rows, cols] f32 tensor: per 32 values
    d = amax / 127 (stored as f16), q = round(x * (1 / d)) with ties away from zero; the packed bytes
    [rows, cols / 32 * 34]."""
    rows, cols = x.shape
    xb = x.view(rows, cols // QK8_0, QK8_0)
    d = xb.abs().amax(-1) / 127.0
    inv = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
    v = xb * inv.unsqueeze(-1)
    q = (torch.sign(v) * torch.floor(v.abs() + 0.5)).to(torch.int8)
    out = torch.empty(rows, cols // QK8_0, 2 + QK8_0, dtype=torch.uint8, device=x.device)
    out[:, :, 0:2] = d.to(torch.float16).view(torch.uint8).view(rows, cols // QK8_0, 2)
    out[:, :, 2:] = q.view(torch.uint8)
    return out.view(rows, -1)


def make_weights(torch, cfg: Qwen2Config, seed: int) -> dict:
    """Random-init weights on the GPU: {'layers': [{wq, wk, wv, wo, wg, wu, wd, attn_norm,
    ffn_norm}], 'final_norm', 'table'}, with cfg.qk_norm also q_norm and k_norm in each layer; linears packed
    Q8_0 (uint8), norms as bf16 bit patterns (int16 tensors)."""
    assert cfg.wtype == Q8_0
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def linear(n, k):
        return quantize_q8_0(torch, torch.randn(n, k, device="cuda", generator=gen) * 0.02).contiguous()

    def norm(n=cfg.hidden):
        w = (1.0 + 0.1 * torch.randn(n, device="cuda", generator=gen)).to(torch.bfloat16)
        return w.view(torch.int16).contiguous()

    H, F = cfg.hidden, cfg.ffn
    layers = []
    for _ in range(cfg.layers):
        layers.append({"wq": linear(cfg.q_dim, H), "wk": linear(cfg.kv_dim, H), "wv": linear(cfg.kv_dim, H),
                       "wo": linear(H, cfg.q_dim), "wg": linear(F, H), "wu": linear(F, H), "wd": linear(H, F),
                       "attn_norm": norm(), "ffn_norm": norm()})
        if cfg.qk_norm:
            layers[-1].update(q_norm=norm(cfg.head_dim), k_norm=norm(cfg.head_dim))
    return {"layers": layers, "final_norm": norm(), "table": linear(cfg.vocab, H)}


class Qwen2Decoder:
    """Greedy decoding of one sequence; buffers for prompts of up to max_prompt tokens and max_seq
    positions in all."""

    def __init__(self, torch, cfg: Qwen2Config, weights: dict, max_seq: int = 512, max_prompt: int = 64,
                 fuse: bool = True):
        self.torch, self.cfg, self.w = torch, cfg, weights
        self.max_seq, self.max_prompt = max_seq, max_prompt
        # decode steps: each RMSNorm inside the launch of the linear that consumes it (the matrix-core
        # decode kernels take in_dim in whole 128-weight chunks for Q8_0), and the rotary embedding with
        # the cache store inside the attention launch
        self.fuse = fuse and cfg.hidden % 128 == 0
        dev, f32, i32 = "cuda", torch.float32, torch.int32
        H, F, P = cfg.hidden, cfg.ffn, max_prompt
        self.rb_h = qlin.row_bytes(cfg.wtype, H)
        self.rb_q = qlin.row_bytes(cfg.wtype, cfg.q_dim)
        self.rb_f = qlin.row_bytes(cfg.wtype, F)
        self.h = torch.zeros(P, H, dtype=f32, device=dev)        # residual stream
        self.xn = torch.zeros(P, H, dtype=f32, device=dev)
        self.q = torch.zeros(P, cfg.q_dim, dtype=f32, device=dev)
        self.k = torch.zeros(P, cfg.kv_dim, dtype=f32, device=dev)
        self.v = torch.zeros(P, cfg.kv_dim, dtype=f32, device=dev)
        self.attn = torch.zeros(P, cfg.q_dim, dtype=f32, device=dev)
        self.act = torch.zeros(P, F, dtype=f32, device=dev)
        self.logits = torch.zeros(cfg.vocab, dtype=f32, device=dev)
        self.pick_scratch = torch.zeros(8192, dtype=torch.uint8, device=dev)  # the head's per-workgroup picks
        f32_caches = 0 if cfg.kv8 else cfg.layers
        self.kc = [torch.zeros(max_seq, cfg.kv_dim, dtype=f32, device=dev) for _ in range(f32_caches)]
        self.vc = [torch.zeros(max_seq, cfg.kv_dim, dtype=f32, device=dev) for _ in range(f32_caches)]
        self.prompt_ids = torch.zeros(P, dtype=i32, device=dev)
        self.token = torch.zeros(1, dtype=i32, device=dev)      # the next step's input token
        self.pos = torch.zeros(1, dtype=i32, device=dev)        # the next step's position
        self.at = torch.zeros(1, dtype=i32, device=dev)         # where a step is taken: past the last position, there
        self.zero = torch.zeros(1, dtype=i32, device=dev)
        self.room = torch.zeros(1, dtype=i32, device=dev)       # drafts that a step by drafts checks
        self.before = torch.zeros(1, dtype=i32, device=dev)     # rows of a step by drafts ahead of the one that completes a block
        self.L = qlin.lib()
        self.controls, self.captured = None, []
        self.adapters = None
        self.stream, self.controlled_on = None, set()  # the calls' stream, and those whose picks read the controls
        if cfg.qk_norm or cfg.kv8:
            qlin.set_stream(torch.cuda.current_stream())
            rows = -(-max_seq // qlin.KV8_BLOCK) * qlin.KV8_BLOCK if cfg.kv8 else max_seq  # (the cache's whole blocks)
            self.rotation = torch.empty(rows, cfg.head_dim, dtype=f32, device=dev)
            qlin.rope_table(self.rotation, cfg.theta)
            norms = [(W["q_norm"], W["k_norm"]) if cfg.qk_norm else (None, None) for W in weights["layers"]]
            self.how = [qlin.QkRope(q, k, 0, cfg.eps, 0, self.rotation, cfg.head_dim) for q, k in norms]
        if cfg.kv8:
            self.kv8 = [qlin.Kv8Cache.empty(torch, 1, cfg.kv_heads, cfg.head_dim, max_seq) for _ in range(cfg.layers)]
            need = max(qlin.attend_kv8_workspace_bytes(1, rows, cfg.n_heads, cfg.kv_heads, cfg.head_dim,
                                                       self.kv8[0].blocks_per_seq) for rows in range(1, P + 1))
            self.attend_ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)

    def set_controls(self, repetition=1.0, frequency=0.0, presence=0.0, bias=None, mask=None) -> None:
        """From the next pick on: penalties for the tokens of the prompt and those picked since (call it before the prefill;
        tokens that came before the first call are not counted), a bias {token: value} of up to 4096 tokens, and a mask
        (int32 words, 32 tokens each, a bit set for a token that may follow; the tensor is read at every pick, so a grammar
        rewrites it between steps).  A graph keeps the controls that it was captured with; what one without controls picks is
        not counted."""
        torch, c = self.torch, self.cfg
        if not repetition > 0:
            raise ValueError(f"repetition {repetition}: must be above 0")
        if mask is not None and (mask.dtype != torch.int32 or tuple(mask.shape) != (1, (c.vocab + 31) // 32)
                                 or not mask.is_contiguous() or mask.device != self.token.device):
            raise ValueError(f"mask: contiguous int32 [1, {(c.vocab + 31) // 32}] on the decoder's device")
        if bias and len(bias) > qlin.MAX_BIAS:
            raise ValueError(f"{len(bias)} biases: at most {qlin.MAX_BIAS}")
        one = lambda v: torch.full((1,), float(v), dtype=torch.float32, device="cuda")
        if self.controls is None:
            self.history = torch.full((1, self.max_seq), -1, dtype=torch.int32, device="cuda")
            self.history_len = torch.zeros(1, dtype=torch.int32, device="cuda")
            self.controlled = torch.zeros(1, c.vocab, dtype=torch.float32, device="cuda")
            self.controls_scratch = torch.empty(max(16, qlin.logits_controls_scratch_bytes(1, c.vocab)), dtype=torch.uint8,
                                                device="cuda")
        if self.controls is not None:
            # picks on other streams than the tensors' own may still have to read them
            for t in self.controls.values():
                for stream in self.controlled_on if t is not None else ():
                    t.record_stream(stream)
            self.controlled_on.clear()
        self.controls = dict(repetition=one(repetition), frequency=one(frequency), presence=one(presence), mask=mask)
        if bias:
            self.controls.update(
                bias_ids=torch.tensor([list(bias)], dtype=torch.int32, device="cuda"),
                bias_values=torch.tensor([list(bias.values())], dtype=torch.float32, device="cuda"))

    LINEARS = (("wq", "wk", "wv"), ("wo",), ("wd",))  # that can have adapters, as they read the same input

    def set_adapters(self, layers, slot, ranks=None, scales=None) -> None:
        """From the next call on: low-rank adapters beside the linears.  layers: for each layer a dict with a qlin.Lora for any of
        wq, wk, wv (of one type, number of slots and rank), wo and wd; slot: the one to use (a number, rewritten by another
        call, or an int32 tensor [1] on the device, which a graph reads at each replay; < 0: none).  ranks int32 and scales
        float32 of the slots, or None.  None instead of layers: no adapters."""
        torch, c = self.torch, self.cfg
        if self.adapters is not None:
            torch.cuda.synchronize()  # (steps on other streams may still read those before)
        if layers is None:
            self.adapters = None
            return
        if len(layers) != c.layers:
            raise ValueError(f"adapters for {len(layers)} layers of {c.layers}")
        dims = {"wq": (c.hidden, c.q_dim), "wk": (c.hidden, c.kv_dim), "wv": (c.hidden, c.kv_dim), "wo": (c.q_dim, c.hidden),
                "wd": (c.ffn, c.hidden)}
        forms = set()
        for L in layers:
            for name, w in L.items():
                if name not in dims or (w.in_dim, w.out_dim) != dims[name]:
                    raise ValueError(f"an adapter {name} of {w.in_dim} to {w.out_dim}")
            for names in self.LINEARS:
                there = [L[n] for n in names if n in L]
                if any(w.like != there[0].like for w in there):
                    raise ValueError("the adapters of wq, wk and wv have one type, number of slots and rank")
                forms.update((len(there), *w.like[1:]) for w in there[:1])
        # (also for fewer rows, which can take more workspace)
        need = max([16] + [qlin.lora_workspace_bytes(rows, *form) for form in forms for rows in range(1, self.max_prompt + 1)])
        ids = torch.empty(self.max_prompt, dtype=torch.int32, device="cuda")
        if not torch.is_tensor(slot):
            slot = torch.full((1,), slot, dtype=torch.int32, device="cuda")
        elif slot.dtype != torch.int32 or slot.numel() != 1 or slot.device != ids.device:
            raise ValueError("slot: a number, or int32 [1] on the decoder's device")
        self.adapters = dict(layers=layers, slot=slot, ids=ids, ranks=ranks, scales=scales,
                             ws=torch.empty(need, dtype=torch.uint8, device="cuda"))
        # (a call on another stream than this one waits for nothing here: the slot is written, and what had the memory before is done)
        torch.cuda.current_stream().synchronize()

    def _adapt(self, layer, x, rows, outs):
        """Adds the layer's adapters of the linears in outs (name: output), which read x."""
        A = self.adapters
        mats = [(A["layers"][layer][n], y[:rows]) for n, y in outs.items() if n in A["layers"][layer]]
        if mats:
            qlin.lora_add(x[:rows], A["ids"], [(w, y, y) for w, y in mats], ranks=A["ranks"], scales=A["scales"], workspace=A["ws"])

    # ---- the calls -------------------------------------------------------------------------------

    def _ok(self, name, rc):
        if rc != 0:
            raise qlin.QlinError(name, rc)

    def _norm(self, x, out, w, rows):
        c = self.cfg
        self._ok("rms_norm", self.L.qlin_launch_rms_norm(x, out, w.data_ptr(), 0, rows, c.hidden, c.eps, 0))

    def _layers(self, rows: int, pos_ptr: int, before: int = 0):
        """The decoder layers over `rows` tokens whose first position is *pos_ptr.  before (an address): the first *before rows
        see the 8-bit cache as it is without the rows after them."""
        c, L, t = self.cfg, self.L, c_ptr
        H, F, QD, KD = c.hidden, c.ffn, c.q_dim, c.kv_dim
        h, xn, q, k, v, attn, act = (t(self.h), t(self.xn), t(self.q), t(self.k), t(self.v), t(self.attn),
                                     t(self.act))
        A = self.adapters
        if A is not None:
            # (the slot stands on the device: captured with what follows)
            A["ids"].copy_(A["slot"].expand(self.max_prompt))
            if self.torch.cuda.is_current_stream_capturing():
                self.captured.append(A)  # (the graph reads these tensors)
        for i, W in enumerate(self.w["layers"]):
            # (adapters of q, k and v read the normed rows, which the fused launch does not write)
            fuse = rows == 1 and self.fuse
            seen = A is not None and any(name in A["layers"][i] for name in self.LINEARS[0])
            if fuse and not seen:
                qlin.rms_norm_quant_gemv_multi(c.wtype, [W["wq"], W["wk"], W["wv"]], self.rb_h, h, W["attn_norm"], 0,
                                               c.eps, 0, [q, k, v], [QD, KD, KD], H)
            elif rows == 1:
                self._norm(h, xn, W["attn_norm"], rows)
                qlin.quant_gemv_multi(c.wtype, [W["wq"], W["wk"], W["wv"]], self.rb_h, xn, [q, k, v], [QD, KD, KD], H)
            else:
                self._norm(h, xn, W["attn_norm"], rows)
                for name, y, n in (("wq", q, QD), ("wk", k, KD), ("wv", v, KD)):
                    self._ok("matmul", L.qlin_launch_quant_matmul(c.wtype, t(W[name]), self.rb_h, xn, y, n, H, rows))
            if seen:
                self._adapt(i, self.xn, rows, {"wq": self.q, "wk": self.k, "wv": self.v})
            if c.kv8:
                qlin.qk_norm_rope_store_kv8(self.how[i], self.kv8[i], q, QD, k, KD, v, KD, q, rows, c.n_heads, pos_ptr)
                qlin.attend_kv8(self.kv8[i], q, attn, rows, c.n_heads, pos_ptr, None, c.head_dim ** -0.5, self.attend_ws)
                if before:  # (once more, in a cache that ends with them: their block is open there)
                    qlin.attend_kv8(self.kv8[i], q, attn, rows, c.n_heads, pos_ptr, before, c.head_dim ** -0.5, self.attend_ws)
            elif c.qk_norm:
                qlin.qk_norm_rope_store_kv(self.how[i], q, QD, k, KD, v, KD, q, self.kc[i], self.vc[i], rows, c.n_heads,
                                           c.kv_heads, c.head_dim, self.max_seq, pos_ptr)
                self._ok("attend", L.qlin_launch_attend(q, t(self.kc[i]), t(self.vc[i]), attn, rows, c.n_heads,
                                                        c.kv_heads, c.head_dim, self.max_seq, pos_ptr))
            elif fuse:
                self._ok("rope_attend", L.qlin_launch_rope_attend(q, k, v, t(self.kc[i]), t(self.vc[i]), attn,
                                                                  c.n_heads, c.kv_heads, c.head_dim, self.max_seq,
                                                                  pos_ptr, c.theta))
            else:
                self._ok("rope", L.qlin_launch_rope_store_kv(q, k, v, t(self.kc[i]), t(self.vc[i]), rows, c.n_heads,
                                                             c.kv_heads, c.head_dim, self.max_seq, pos_ptr, c.theta))
                self._ok("attend", L.qlin_launch_attend(q, t(self.kc[i]), t(self.vc[i]), attn, rows, c.n_heads,
                                                        c.kv_heads, c.head_dim, self.max_seq, pos_ptr))
            self._ok("o", L.qlin_launch_quant_matmul_add(c.wtype, t(W["wo"]), self.rb_q, attn, h, H, QD, rows))
            if A is not None:
                self._adapt(i, self.attn, rows, {"wo": self.h})
            if fuse:  # (its gate and up have no adapters)
                self._ok("norm_swiglu", L.qlin_launch_rms_norm_quant_swiglu(c.wtype, t(W["wg"]), t(W["wu"]), self.rb_h,
                                                                            h, t(W["ffn_norm"]), 0, c.eps, 0, act, F,
                                                                            H))
            elif rows == 1:
                self._norm(h, xn, W["ffn_norm"], rows)
                self._ok("swiglu", L.qlin_launch_quant_swiglu(c.wtype, t(W["wg"]), t(W["wu"]), self.rb_h, self.rb_h,
                                                              xn, act, F, H))
            else:
                self._norm(h, xn, W["ffn_norm"], rows)
                self._ok("swiglu", L.qlin_launch_quant_swiglu_rows(c.wtype, t(W["wg"]), t(W["wu"]), self.rb_h,
                                                                   self.rb_h, xn, act, F, H, rows))
            self._ok("down", L.qlin_launch_quant_matmul_add(c.wtype, t(W["wd"]), self.rb_f, act, h, H, F, rows))
            if A is not None:
                self._adapt(i, self.act, rows, {"wd": self.h})

    def _head(self, row: int):
        """Final norm of residual row `row`, the tied output head, and the greedy pick into token."""
        c, L, t = self.cfg, self.L, c_ptr
        hr = t(self.h) + 4 * row * c.hidden
        if self.controls is not None:
            if self.torch.cuda.is_current_stream_capturing():
                self.captured.append(self.controls)  # (the graph reads these tensors)
            else:
                self.controlled_on.add(self.stream)
            if self.fuse and hr % 16 == 0:
                qlin.rms_norm_quant_gemv_multi(c.wtype, [self.w["table"]], self.rb_h, hr, self.w["final_norm"], 0, c.eps, 0,
                                               [self.logits], [c.vocab], c.hidden)
            else:
                self._norm(hr, t(self.xn), self.w["final_norm"], 1)
                self._ok("lm_head", L.qlin_launch_quant_gemv(c.wtype, t(self.w["table"]), self.rb_h, t(self.xn),
                                                             t(self.logits), c.vocab, c.hidden, 1))
            qlin.logits_controls(self.logits.view(1, -1), self.controlled, 1, c.vocab, history=self.history,
                                 history_lens=self.history_len, picks=self.token, scratch=self.controls_scratch,
                                 **self.controls)
            return
        if self.fuse and hr % 16 == 0:
            # the norm inside the head GEMV, and each of its workgroups' greedy pick in its epilogue (one
            # small launch reduces the picks): two launches instead of norm, GEMV and a scan of every logit
            self._ok("lm_head_argmax", L.qlin_launch_quant_gemv_argmax(
                c.wtype, t(self.w["table"]), self.rb_h, hr, t(self.w["final_norm"]), 0, c.eps, 0, t(self.logits),
                c.vocab, c.hidden, t(self.pick_scratch), t(self.token)))
            return
        self._norm(hr, t(self.xn), self.w["final_norm"], 1)
        self._ok("lm_head", L.qlin_launch_quant_gemv(c.wtype, t(self.w["table"]), self.rb_h, t(self.xn),
                                                     t(self.logits), c.vocab, c.hidden, 1))
        self._ok("argmax", L.qlin_launch_argmax(t(self.logits), c.vocab, t(self.token)))

    def prefill(self, prompt) -> None:
        """The prompt (device int32 tensor of n <= max_prompt ids) at positions 0..n-1 in one batched
        pass; leaves the last position's logits, the greedy token and pos = n."""
        c, t = self.cfg, c_ptr
        n = int(prompt.numel())
        assert 0 < n <= self.max_prompt and n <= self.max_seq
        self.stream = self.torch.cuda.current_stream()
        qlin.set_stream(self.stream)
        self.prompt_ids[:n].copy_(prompt)
        self._ok("embedding", self.L.qlin_launch_quant_embedding(c.wtype, t(self.prompt_ids), t(self.h),
                                                                 t(self.w["table"]), self.rb_h, c.hidden, n))
        self._layers(n, t(self.zero))
        if self.controls is not None:
            self.history.fill_(-1)  # (steps of a graph without controls leave rows between: no tokens of another text)
            self.history[0, :n].copy_(prompt)
            self.history_len.fill_(n)
        self._head(n - 1)
        self.pos.fill_(n)

    def step(self) -> None:
        """One decode token: the token id and position held on the device; leaves the logits, the next
        greedy token and pos + 1 (no host synchronisation, so a HIP graph can hold it)."""
        c, t = self.cfg, c_ptr
        self.stream = self.torch.cuda.current_stream()
        qlin.set_stream(self.stream)
        self._ok("embedding", self.L.qlin_launch_quant_embedding(c.wtype, t(self.token), t(self.h),
                                                                 t(self.w["table"]), self.rb_h, c.hidden, 1))
        if c.kv8 or self.controls is not None:
            # past the last position that one is taken again, as the f32 caches' launches do by themselves
            self.torch.clamp(self.pos, max=self.max_seq - 1, out=self.at)
        self._layers(1, t(self.at if c.kv8 else self.pos))
        if self.controls is not None:
            # the step's token is history for its pick
            self.history[0].scatter_(0, self.at.long(), self.token)
            self.torch.add(self.pos, 1, out=self.history_len)
        self._head(0)
        self.pos.add_(1)

    def drafts(self, n: int) -> dict:
        """What a call of step_drafts with n drafted tokens works on, for as long as it is used: drafts int32 [1, n] and
        uniform float32 [1, n + 1] (numbers in [0, 1)), which the caller fills, and n_drafts int32 [1] (at first n) and
        temperature float32 [1] (at first 0: greedy); tokens int32 [1, n + 1] (-1 after the last), accepted int32 [1], logprobs
        and rates, which the call fills."""
        torch, c, dev = self.torch, self.cfg, "cuda"
        if not 0 <= n < min(self.max_prompt, qlin.KV8_BLOCK):  # (as far as the 8-bit cache takes positions back)
            raise ValueError(f"{n} drafted tokens: at most {min(self.max_prompt, qlin.KV8_BLOCK) - 1}")
        f = lambda *shape: torch.zeros(*shape, dtype=torch.float32, device=dev)
        i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=dev)
        d = dict(drafts=i(1, n), uniform=f(1, n + 1), n_drafts=torch.full((1,), n, dtype=torch.int32, device=dev), temperature=f(1),
                 tokens=i(1, n + 1), accepted=i(1), logprobs=f(1, n + 1), rates=f(1, n), logits=f(1, n + 1, c.vocab),
                 ws=torch.empty(max(16, qlin.verify_drafts_workspace_bytes(1, n, c.vocab)), dtype=torch.uint8, device=dev))
        torch.cuda.current_stream().synchronize()  # (as set_adapters)
        return d

    def step_drafts(self, d: dict, draft_logits=None) -> None:
        """Decode tokens by drafts (of self.drafts(n)): the next token and the n drafted ones after it in one pass, those
        that the model's probabilities accept and one more; leaves pos after them and the last one as the next token (no host
        synchronisation).  A row's logits (d["logits"]) depend on no draft after it.  draft_logits float32 [1, n, vocab], or
        None for drafts by lookup.  Drafts that the cache has no position for are not checked, as if n_drafts left them out; from
        the last position on that one is taken again, as step() does.  Controls of the pick do not go with it."""
        c, t, torch = self.cfg, c_ptr, self.torch
        if self.controls is not None:
            raise ValueError("drafts are not checked under controls")
        rows = d["tokens"].shape[1]
        self.stream = torch.cuda.current_stream()
        qlin.set_stream(self.stream)
        self.prompt_ids[:1].copy_(self.token)
        # (a draft past n_drafts may be anything)
        self.prompt_ids[1:rows].copy_(d["drafts"][0].clamp(0, c.vocab - 1))
        self._ok("embedding", self.L.qlin_launch_quant_embedding(c.wtype, t(self.prompt_ids), t(self.h), t(self.w["table"]),
                                                                 self.rb_h, c.hidden, rows))
        # (drafts that there are positions for: the room is on the device, as the position is)
        torch.clamp(self.pos, max=self.max_seq - 1, out=self.at)
        torch.minimum(d["n_drafts"], (self.max_seq - 1) - self.at, out=self.room)
        before = 0
        if c.kv8 and rows > 1:
            # A block that ends at row b stands in codes, whose scale has all of its rows, also drafts that may be rejected: the
            # rows before b see it as it was, open.  (At most 32 rows: one block ends among them, or none.)
            torch.bitwise_and(torch.bitwise_not(self.at), qlin.KV8_BLOCK - 1, out=self.before)
            self.before.masked_fill_(self.before >= rows, 0)
            before = t(self.before)
        self._layers(rows, t(self.at), before)
        self._norm(t(self.h), t(self.xn), self.w["final_norm"], rows)
        self._ok("lm_head", self.L.qlin_launch_quant_matmul(c.wtype, t(self.w["table"]), self.rb_h, t(self.xn), t(d["logits"]),
                                                            c.vocab, c.hidden, rows))
        qlin.verify_drafts(d["logits"], d["drafts"], d["uniform"], d["tokens"], d["accepted"], draft_logits=draft_logits,
                           n_drafts=self.room, temperature=d["temperature"], logprobs=d["logprobs"], rates=d["rates"],
                           workspace=d["ws"])
        torch.index_select(d["tokens"][0], 0, d["accepted"], out=self.token)
        self.pos.add_(d["accepted"]).add_(1)

    def generate(self, prompt, n_new: int, logits_out=None):
        """Greedy decode of n_new tokens after the prompt, eagerly; returns the token ids (host list).
        logits_out ([n_new, vocab] device tensor, optional) receives each new token's logits."""
        torch = self.torch
        toks = torch.zeros(n_new, dtype=torch.int32, device="cuda")
        self.prefill(prompt)
        for i in range(n_new):
            if i:
                self.step()
            toks[i:i + 1].copy_(self.token)
            if logits_out is not None:
                logits_out[i].copy_(self.logits)
        return toks.cpu().tolist()


def c_ptr(t) -> int:
    return t.data_ptr()
