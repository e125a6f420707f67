"""Language-model training step built on the FirstPassageAttention layer (the reference's README describes this
model; the reference repository ships only the layer, kernel.py:512-530).

The model is a GPT-2-small-shaped decoder: token embedding (no positional embedding: FPA's field carries order),
`n_layers` pre-LayerNorm blocks of FirstPassageAttention and a 4x GELU MLP, a final LayerNorm and an output layer
tied to the embedding. Each block's field is the layer's own: per head delta, g, h are linear maps of x,
W = cumsum(delta), phi = W + g, psi = W + h, beta = softplus(beta_raw).

`LMTrainer.step` runs one optimisation step: fp16 autocast forward, cross-entropy of the next token, loss scaling
(torch.amp.GradScaler), backward, AdamW. Under torch.distributed the model is wrapped in DistributedDataParallel,
whose gradient all-reduce runs over NCCL.

`LMGenerator` answers with a trained model on a CUDA device: a paged cache for each layer (int8 or not), prompts behind
a prefix that the whole batch shares, and drafted tokens verified against the model's probabilities.
"""
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from .ops import FirstPassageAttention, first_passage_attention
from .serving import MAX_NEW_TOKENS, FPACache, first_passage_decode, verify_draft


@dataclass
class LMConfig:
    vocab: int = 50304
    d_model: int = 768
    n_heads: int = 12
    n_layers: int = 12
    tau: float = 1.0
    beta_init: float = 1.0


class MLP(nn.Module):
    def __init__(self, d_model):
        super().__init__()
        self.fc = nn.Linear(d_model, 4 * d_model)
        self.proj = nn.Linear(4 * d_model, d_model)

    def forward(self, x):
        return self.proj(F.gelu(self.fc(x), approximate="tanh"))


class Block(nn.Module):
    def __init__(self, cfg, impl):
        super().__init__()
        self.ln1 = nn.LayerNorm(cfg.d_model)
        self.attn = FirstPassageAttention(cfg.d_model, cfg.n_heads, tau=cfg.tau, beta_init=cfg.beta_init, impl=impl)
        self.ln2 = nn.LayerNorm(cfg.d_model)
        self.mlp = MLP(cfg.d_model)

    def forward(self, x):
        x = x + self.attn(self.ln1(x))
        return x + self.mlp(self.ln2(x))


class FPALanguageModel(nn.Module):
    def __init__(self, cfg=LMConfig(), impl=None):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab, cfg.d_model)
        self.blocks = nn.ModuleList(Block(cfg, impl) for _ in range(cfg.n_layers))
        self.ln_f = nn.LayerNorm(cfg.d_model)
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, std=0.02)
            if m.bias is not None:
                nn.init.zeros_(m.bias)
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, std=0.02)

    def forward(self, idx):
        x = self.wte(idx)
        for blk in self.blocks:
            x = blk(x)
        return F.linear(self.ln_f(x), self.wte.weight)  # output layer tied to the embedding

    def n_params(self):
        return sum(p.numel() for p in self.parameters())


def make_tokens(batch, T, vocab, seed, device):
    """Token ids uniform over the vocabulary, [batch, T + 1] (inputs and next-token targets)."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randint(0, vocab, (batch, T + 1), generator=g).to(device)


class LMTrainer:
    """One training step per call: fp16 autocast, next-token cross-entropy, GradScaler, AdamW; DDP when the
    default process group is initialised with more than one rank."""

    def __init__(self, model, lr=3e-4, weight_decay=0.1, ddp=None):
        self.model = model
        if ddp is None:
            ddp = torch.distributed.is_available() and torch.distributed.is_initialized() and \
                torch.distributed.get_world_size() > 1
        if ddp:
            dev = next(model.parameters()).device
            self.net = nn.parallel.DistributedDataParallel(model, device_ids=[dev.index] if dev.type == "cuda" else None)
        else:
            self.net = model
        dev_type = next(model.parameters()).device.type
        self.opt = torch.optim.AdamW(model.parameters(), lr=lr, weight_decay=weight_decay, betas=(0.9, 0.95),
                                     fused=dev_type == "cuda")
        self.amp = dev_type == "cuda"
        self.scaler = torch.amp.GradScaler("cuda", enabled=self.amp)

    def loss(self, tokens):
        inp, tgt = tokens[:, :-1], tokens[:, 1:]
        with torch.autocast(device_type="cuda", dtype=torch.float16, enabled=self.amp):
            logits = self.net(inp)
        return F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), tgt.reshape(-1))

    def step(self, tokens):
        """One optimisation step; returns the loss (a 0-d tensor on the model's device, not synchronised)."""
        loss = self.loss(tokens)
        self.scaler.scale(loss).backward()
        self.scaler.step(self.opt)
        self.scaler.update()
        self.opt.zero_grad(set_to_none=True)
        return loss.detach()


class LMGenerator:
    """Serves an FPALanguageModel: one FPACache per layer over common block tables, and the field's walk at the end of
    every sequence.

    `extend(tokens)` runs the next n tokens of every sequence (at most 16 at a time after the first chunk) and returns
    their logits; `keep(counts)` says how many of them stay (refused drafts, or the padding of a ragged batch, are
    simply written over by the next call). Tokens that `reset` made no room for are refused. `generate` samples with or
    without a draft model, and raises what the kernels recorded in the caches' status words.

    dtype float16 runs the model under fp16 autocast, as training does, on the tensor-core kernels; float32 runs it as it
    is. storage=torch.int8 quantises the caches."""

    def __init__(self, model, max_tokens, page_size=64, dtype=torch.float16, storage=None):
        cfg, dev = model.cfg, next(model.parameters()).device
        self.model, self.dtype, self.page, self.device = model.eval(), dtype, page_size, dev
        self.n_pages = -(-max_tokens // page_size)
        self.caches = [FPACache(self.n_pages, cfg.n_heads, cfg.d_model // cfg.n_heads, page_size, dtype, storage, dev)
                       for _ in range(cfg.n_layers)]
        self.reset(0, 0)

    def reset(self, batch, tokens, prefix=None):
        """Start `batch` empty sequences with room for `tokens` tokens each, behind the tokens of `prefix` (a list, run
        once here) if given."""
        cfg = self.model.cfg
        self._check_ids(prefix or [])
        per, n_pre = max(-(-tokens // self.page), 1), 0 if prefix is None else -(-len(prefix) // self.page)
        if n_pre + batch * per > self.n_pages:
            raise ValueError(f"the cache has {self.n_pages} pages, {n_pre + batch * per} are needed")
        i32 = dict(dtype=torch.int32, device=self.device)
        self.prefix, self._most = {}, 0  # _most: no sequence is longer (the lengths are on the device)
        if n_pre:
            self.table = torch.arange(n_pre, **i32)[None]
            self.lengths, self.walk = torch.zeros(1, **i32), torch.zeros(cfg.n_layers, 1, cfg.n_heads, device=self.device)
            self.extend(torch.tensor([list(prefix)], device=self.device), first=True, logits=False)
            self.keep(torch.tensor([len(prefix)], **i32))
            walk, table = self.walk, self.table[0]
            self.prefix = dict(prefix_table=table, prefix_len=len(prefix))
        self.table = n_pre + torch.arange(batch * per, **i32).view(batch, per)
        self.lengths, self._most = torch.zeros(batch, **i32), 0
        self.walk = walk.expand(-1, batch, -1).contiguous() if n_pre else \
            torch.zeros(cfg.n_layers, batch, cfg.n_heads, device=self.device)

    def _check_ids(self, ids):
        # On the device an id outside the embedding is a fault that ends the process.
        if any(not 0 <= t < self.model.cfg.vocab for t in ids):
            raise ValueError(f"token ids must lie in [0, {self.model.cfg.vocab})")

    def _field(self, field, x, walk):
        """The layer's field of the next tokens (`Field` starts its walk at 0): phi, psi [B, H, n], and the walk
        [B, n, H] after each of them."""
        B, n, _ = x.shape
        with torch.autocast(device_type="cuda", enabled=False):
            out = F.linear(x.float(), field.proj.weight.float(), field.proj.bias.float()).view(B, n, 3, -1)
            w = walk[:, None] + out[:, :, 0].cumsum(1)
            return (w + out[:, :, 1]).transpose(1, 2), (w + out[:, :, 2]).transpose(1, 2), w

    @torch.no_grad()
    def extend(self, tokens, first=False, logits=True):
        """Logits [B, n, vocab] of the next tokens [B, n] of every sequence, which enter the caches at `lengths`.
        first: the sequences are empty and there is no prefix; n may then exceed 16, and the tokens attend to each
        other through the training kernels. logits False: fill the caches only, and return None."""
        m, (B, n) = self.model, tokens.shape
        if n > MAX_NEW_TOKENS and not first:
            raise ValueError(f"at most {MAX_NEW_TOKENS} tokens at a time")
        room = self.table.shape[1] * self.page
        if self._most + n > room or (first and self._most):
            self._most = max(self.lengths.tolist(), default=0)  # waits for the device, when the bound is no longer enough
        if self._most + n > room:
            raise ValueError(f"{n} tokens after {self._most} exceed the room of {room} tokens")
        if first and (self._most or self.prefix):
            raise ValueError("first: only for empty sequences without a prefix")
        upto, walks = self.lengths + n, []
        with torch.autocast(device_type="cuda", dtype=torch.float16, enabled=self.dtype == torch.float16):
            x = m.wte(tokens)
            for layer, (blk, cache) in enumerate(zip(m.blocks, self.caches)):
                y, at = blk.ln1(x), blk.attn
                q, k, v = at.qkv(y).view(B, n, 3, at.h, at.d).permute(2, 0, 3, 1, 4)
                phi, psi, w = self._field(at.field, y, self.walk[layer])
                beta = F.softplus(at.field.beta_raw).float()
                cache.append(k, v, phi, psi, self.table, self.lengths)
                if first:
                    o = first_passage_attention(q, k, v, phi, psi, beta)
                else:
                    o = first_passage_decode(q, cache, self.table, upto, beta, **self.prefix)
                x = x + at.out(o.transpose(1, 2).reshape(B, n, -1))
                x = x + blk.mlp(blk.ln2(x))
                walks.append(w)
            self._walks = torch.stack(walks)  # [layers, B, n, H]
            return F.linear(m.ln_f(x), m.wte.weight).float() if logits else None

    def keep(self, counts):
        """The first counts[b] (int32) of the tokens of the last `extend` stay; at most all of them."""
        counts = counts.clamp(0, self._walks.shape[2])
        self._most += self._walks.shape[2]
        self.lengths = self.lengths + counts
        w = torch.cat([self.walk[:, :, None], self._walks], 2)
        self.walk = w.gather(2, counts.long()[None, :, None, None].expand(w.shape[0], -1, 1, w.shape[3]))[:, :, 0]

    def _start(self, prompts, room, prefix):
        """Run the prompts but for their last tokens, which the caller feeds next."""
        self.reset(len(prompts), max(len(p) for p in prompts) + room, prefix)
        lens = torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device=self.device)
        T = max(len(p) for p in prompts) - 1
        padded = torch.tensor([list(p[:-1]) + [0] * (T - len(p) + 1) for p in prompts], device=self.device)
        if T and not self.prefix:
            self.extend(padded, first=True, logits=False)
            self.keep(lens)
        elif T:
            for i in range(0, T, MAX_NEW_TOKENS):
                part = padded[:, i:i + MAX_NEW_TOKENS]
                self.extend(part, logits=False)
                self.keep((lens - i).clamp(0, part.shape[1]).int())
        return torch.tensor([p[-1] for p in prompts], device=self.device)

    @torch.no_grad()
    def generate(self, prompts, n_new, temperature=1.0, prefix=None, draft=None, n_draft=4, generator=None):
        """n_new sampled tokens after each prompt (lists of token ids, none empty), behind the tokens of `prefix` if
        given. draft: an LMGenerator with a smaller model of the same vocabulary that proposes n_draft tokens (at most
        15) a round; they are accepted so that the samples keep this model's distribution."""
        if draft is None:
            n_draft = 0
        if not 0 <= n_draft < MAX_NEW_TOKENS or any(len(p) == 0 for p in prompts):
            raise ValueError(f"n_draft must lie below {MAX_NEW_TOKENS}, and no prompt may be empty")
        if not prompts:
            raise ValueError("at least one prompt")
        for p in prompts:
            self._check_ids(p)
        if draft is not None and draft.model.cfg.vocab != self.model.cfg.vocab:
            raise ValueError("the draft's vocabulary must be the model's")
        if not temperature > 0:
            raise ValueError("the temperature must be positive")
        if draft is self:
            raise ValueError("the draft needs caches of its own (another LMGenerator; the model may be the same)")
        B, room = len(prompts), n_new + 2 * n_draft + 2
        cur = self._start(prompts, room, prefix)
        if draft is not None:
            draft._start(prompts, room, prefix)
        rand = dict(device=self.device, generator=generator)
        out, done = [[] for _ in prompts], torch.zeros(B, dtype=torch.bool, device=self.device)
        while min(len(x) for x in out) < n_new:
            tokens, q, steps = [cur], [], []
            for _ in range(n_draft):
                probs = (draft.extend(tokens[-1][:, None])[:, 0] / temperature).softmax(-1)
                steps.append((draft.lengths, draft.walk))
                draft.keep(torch.ones_like(draft.lengths))
                q.append(probs)
                tokens.append((probs / torch.empty_like(probs).exponential_(generator=generator)).argmax(-1))
            if n_draft:  # the last draft enters the draft's cache too, in case it is accepted
                draft.extend(tokens[-1][:, None])
                steps.append((draft.lengths, draft.walk))
                draft.keep(torch.ones_like(draft.lengths))
                steps.append((draft.lengths, draft.walk))
            new = torch.stack(tokens, 1)
            p = (self.extend(new) / temperature).softmax(-1)
            noise = torch.empty(B, p.shape[-1], device=self.device).exponential_(generator=generator)
            accepted, picked = verify_draft(p, torch.stack(q, 1) if q else p[:, :0], new[:, 1:], torch.rand(B, n_draft, **rand), noise)
            # A sequence that has all its tokens stays where it is until the others have theirs.
            stay = torch.where(done, 0, accepted + 1)
            self.keep(stay)
            if n_draft:
                # The draft goes back to the state after the tokens that stay.
                at = stay.long()
                draft.lengths = torch.stack([s[0] for s in steps], 1).gather(1, at[:, None])[:, 0]
                walks = torch.stack([s[1] for s in steps], 2)
                draft.walk = walks.gather(2, at[None, :, None, None].expand(walks.shape[0], -1, 1, walks.shape[3]))[:, :, 0]
            cur = torch.where(done, cur, picked.gather(1, accepted.long()[:, None])[:, 0])
            for x, row in zip(out, picked.tolist()):
                if len(x) < n_new:
                    x.extend(t for t in row if t >= 0)
            done = torch.tensor([len(x) >= n_new for x in out], device=self.device)
        for cache in self.caches + (draft.caches if draft is not None else []):
            cache.check()
        return [x[:n_new] for x in out]
