"""Decoding over a paged key-value cache: after the first token, without copying the cache.

The reference decodes by running the HF model over the request's DynamicCache (tread/server.py:200-211),
which concatenates every new token's keys and values to each layer's tensors: the whole cache is
copied for each token, and each request decodes by itself. Here a sequence's keys and values live in
pages of a pool shared by all sequences; a decode step of a batch of sequences of any lengths is, per layer,

    qkv = RMSNorm(h) @ Wqkv^T + b                       (Qwen2Rows.qkv)
    rotate q and k at the row's position, append k, v   (tread_paged_append)
    o = attention of q over the sequence's pages        (tread_paged_attn)
    h = h + o @ Wo^T ; h = h + down(silu(gate) * up)    (Qwen2Rows.layer_tail)

    dec = PagedDecoder(model, num_pages=1024)
    logits, cache, stats = engine.prefill(prefix_ids, docs, query_ids)
    seq = dec.admit(cache)                  # one launch: all layers into pages
    logits = dec.step([seq], [int(logits.argmax())])     # [1, vocab]
    dec.release(seq)
"""
import torch

from tread_b200 import kernels
from tread_b200.blend import rows_of
from tread_b200.graphs import capture


class OutOfPages(RuntimeError):
    """No free page (or no free sequence) is left in the pool."""


class PagedCache:
    """Pools of pages [num_pages, L, Hkv, page_size, D] for K and V, and the page tables of up to
    `max_seqs` sequences of up to `max_len` tokens. The bookkeeping is the host's; the tables are on the
    device, int32 [max_seqs, pages of max_len], entries of pages that a sequence does not hold -1. Made inside
    inference mode or outside of it, it is used in either."""

    def __init__(self, L, Hkv, D, num_pages, page_size=64, max_seqs=64, max_len=32768, dtype=torch.bfloat16,
                 device="cuda"):
        if min(num_pages, page_size, max_seqs, max_len) < 1:
            raise ValueError("num_pages, page_size, max_seqs and max_len must be at least 1")
        shape = (num_pages, L, Hkv, page_size, D)
        self.K = torch.zeros(shape, dtype=dtype, device=device)
        self.V = torch.zeros(shape, dtype=dtype, device=device)
        self.page_size, self.max_seqs, self.max_len = page_size, max_seqs, max_len
        self.table = torch.full((max_seqs, self.pages_of(max_len)), -1, dtype=torch.int32, device=device)
        self.lens = {}  # sequence -> tokens
        self._pages = {}  # sequence -> its pages in order
        self._free = list(range(num_pages - 1, -1, -1))
        self._free_seqs = list(range(max_seqs - 1, -1, -1))

    def pages_of(self, tokens):
        return -(-tokens // self.page_size)

    @property
    def free_pages(self):
        return len(self._free)

    def layer(self, l):
        """The pools of layer l, views [num_pages, Hkv, page_size, D]."""
        return self.K[:, l], self.V[:, l]

    @torch.inference_mode()
    def new(self, tokens=0):
        """A new sequence with room for `tokens` tokens; it holds none yet."""
        if not self._free_seqs:
            raise OutOfPages(f"all {self.max_seqs} sequences are in use")
        seq = self._free_seqs.pop()
        self.lens[seq], self._pages[seq] = 0, []
        try:
            self.reserve(seq, tokens)
        except Exception:
            self.release(seq)
            raise
        return seq

    @torch.inference_mode()
    def reserve(self, seq, tokens):
        """Give `seq` pages for `tokens` tokens in all (nothing changes if that fails)."""
        pages = self._pages[seq]
        if tokens > self.max_len:
            raise ValueError(f"{tokens} tokens, but sequences have at most {self.max_len}")
        need = self.pages_of(tokens) - len(pages)
        if need <= 0:
            return
        if need > len(self._free):
            raise OutOfPages(f"{need} pages wanted, {len(self._free)} free")
        new = [self._free.pop() for _ in range(need)]
        at = len(pages)
        pages.extend(new)
        if need == 1:
            self.table[seq, at].fill_(new[0])
        else:
            self.table[seq, at:at + need] = torch.tensor(new, dtype=torch.int32).to(self.table.device)

    @torch.inference_mode()
    def release(self, seq):
        """Give back the sequence and its pages."""
        if seq not in self.lens:
            raise ValueError(f"release: no sequence {seq}")
        self._free.extend(reversed(self._pages.pop(seq)))
        del self.lens[seq]
        self.table[seq].fill_(-1)
        self._free_seqs.append(seq)


def _flat_layers(layers):
    """The layers' [1, Hkv, T, D] tensors as one view [T, L * Hkv, D] where they are the slices of one
    contiguous [L, 1, Hkv, T, D] tensor (a request cache as the engine hands it out), else None."""
    first = layers[0]
    _, H, T, D = first.shape
    step = H * T * D * first.element_size()
    for l, t in enumerate(layers):
        if (t.shape != first.shape or not t.is_contiguous() or t.data_ptr() != first.data_ptr() + l * step
                or t.untyped_storage().data_ptr() != first.untyped_storage().data_ptr()):
            return None
    return first.as_strided((T, len(layers) * H, D), (D, T * D, 1))


class PagedDecoder:
    """Decode steps of a model (or its rows: Qwen2Rows, TPQwen2Rows) over a PagedCache.

    graphs=True captures one CUDA graph per batch size (powers of two up to `max_seqs`); a step of fewer
    sequences pads the batch with rows of position -1, which append nothing and attend to nothing.

    Used from one stream at a time, as the engine is: the rows' projections share a workspace (eager steps,
    captured ones and other decoders of the same device alike)."""

    def __init__(self, model, num_pages, page_size=64, max_seqs=64, max_len=32768, graphs=False):
        net = self.net = rows_of(model)
        if graphs and getattr(net, "world", 1) > 1:
            raise ValueError("graphs=True is not supported with tensor-parallel rows")
        if net.D not in (64, 128, 256) or net.Hq > 16 * net.Hkv:
            raise ValueError(f"paged attention takes heads of 64, 128 or 256 in groups of up to 16, not of {net.D} in "
                             f"groups of {net.Hq // net.Hkv}")
        self.cache = PagedCache(net.L, net.Hkv, net.D, num_pages, page_size, max_seqs, max_len, net.dtype, net.device)
        self.inv_freq = torch.tensor(net.inv_freq, dtype=torch.float32, device=net.device)
        self.graphs = {} if graphs else None

    @property
    def max_len(self):
        """Tokens that one sequence can have with the whole pool to itself."""
        return min(self.cache.max_len, self.cache.K.shape[0] * self.cache.page_size)

    @torch.inference_mode()
    def admit(self, cache, room=0):
        """A new sequence that starts with a request's cache (the DynamicCache of Engine.prefill, or any with
        per-layer [1, Hkv, T, D] tensors), copied into pages; with pages for `room` further tokens. The
        given cache is not needed afterwards."""
        keys = [layer.keys for layer in cache.layers]
        values = [layer.values for layer in cache.layers]
        if len(keys) != self.net.L:
            raise ValueError(f"admit: a cache of {len(keys)} layers, the model has {self.net.L}")
        T = keys[0].shape[2] if keys[0].dim() == 4 else 0
        want = (1, self.net.Hkv, T, self.net.D)
        for t in keys + values:
            if t.shape != want:
                raise ValueError(f"admit: layers must be [1, {self.net.Hkv}, T, {self.net.D}] of one length, got "
                                 f"{list(t.shape)}")
        pc = self.cache
        seq = pc.new(T + room)
        try:
            pos = torch.arange(T, device=self.net.device)
            table = pc.table[seq:seq + 1]
            of = torch.zeros(T, dtype=torch.int32, device=self.net.device)
            k, v = _flat_layers(keys), _flat_layers(values)
            if k is not None and v is not None:
                kernels.paged_append(k, v, pc.K.flatten(1, 2), pc.V.flatten(1, 2), table, pos, seq=of, err=self.net.err)
            else:
                for l in range(self.net.L):
                    kp, vp = pc.layer(l)
                    kernels.paged_append(keys[l][0].transpose(0, 1), values[l][0].transpose(0, 1), kp, vp, table, pos,
                                         seq=of, err=self.net.err)
        except Exception:
            pc.release(seq)
            raise
        pc.lens[seq] = T
        return seq

    def release(self, seq):
        self.cache.release(seq)

    def _forward(self, tokens, pos, table):
        """Logits [B, vocab] of one new token per row at positions pos, appended to the rows' pages."""
        net = self.net
        B, nq, nk = tokens.shape[0], net.Hq * net.D, net.Hkv * net.D
        lens = (pos + 1).clamp_(min=0)
        h = net.embed_ids(tokens)
        for l in range(net.L):
            qkv = net.qkv(l, h)
            kp, vp = self.cache.layer(l)
            q = kernels.paged_append(qkv[:, nq:nq + nk].unflatten(1, (net.Hkv, net.D)),
                                     qkv[:, nq + nk:].unflatten(1, (net.Hkv, net.D)), kp, vp, table, pos,
                                     inv_freq=self.inv_freq, attn_scaling=net.attn_scaling,
                                     q=qkv[:, :nq].unflatten(1, (net.Hq, net.D)), err=net.err)
            o = kernels.paged_attn(q, kp, vp, table, lens, err=net.err)
            h = net.layer_tail(l, h, o.view(B, nq))
        return net.logits(h)

    def _ids(self, tokens):
        """Token ids [B] as an int64 device tensor, all inside the vocabulary: an embedding lookup outside it is a
        device-side assertion, after which the process has no GPU."""
        net = self.net
        t = torch.as_tensor(tokens)
        if t.dim() != 1 or t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
            raise ValueError(f"step: tokens must be whole numbers, one a sequence, got {t.dtype} {list(t.shape)}")
        vocab = net.embed.shape[0]
        if t.is_cuda:  # not read back: the step runs with the nearest id, and check_errors() raises
            t = t.to(net.device, torch.int64)
            ids = t.clamp(0, vocab - 1)
            net.err[:1].bitwise_or_((ids != t).any().to(torch.int32))
            return ids
        t = t.to(torch.int64)
        if int(t.min()) < 0 or int(t.max()) >= vocab:
            raise ValueError(f"step: token ids from {int(t.min())} to {int(t.max())}, the vocabulary has {vocab}")
        return t.to(net.device)

    @torch.inference_mode()
    def step(self, seqs, tokens):
        """Append tokens[i] to sequence seqs[i] and return the logits of what follows, [len(seqs), vocab].
        seqs: distinct sequences; tokens: their ids, a list or a tensor of whole numbers [len(seqs)]. Ids outside
        the vocabulary are refused; those of a device tensor, which is not read back, are replaced by the nearest
        one, and net.check_errors() raises. Where a sequence's pages do not suffice, nothing happens and
        OutOfPages (or ValueError past max_len) is raised. With graphs the result is the graph's own buffer,
        valid until the next step (a graph serves all batch sizes up to its power of two)."""
        pc, dev = self.cache, self.net.device
        B = len(seqs)
        if B == 0 or len(set(seqs)) != B or not all(s in pc.lens for s in seqs):
            raise ValueError("step: seqs must be distinct sequences of this decoder")
        if len(tokens) != B:
            raise ValueError(f"step: {len(tokens)} tokens for {B} sequences")
        need = [pc.lens[s] + 1 for s in seqs]
        if max(need) > pc.max_len:
            raise ValueError(f"{max(need)} tokens, but sequences have at most {pc.max_len}")
        short = sum(max(0, pc.pages_of(n) - len(pc._pages[s])) for s, n in zip(seqs, need))
        if short > pc.free_pages:
            raise OutOfPages(f"{short} pages wanted, {pc.free_pages} free")
        tokens = self._ids(tokens)
        for s, n in zip(seqs, need):
            pc.reserve(s, n)
        at = torch.tensor([[pc.lens[s] for s in seqs], list(seqs)])
        at = at.pin_memory().to(dev, non_blocking=True) if dev.type == "cuda" else at
        if self.graphs is None:
            logits = self._forward(tokens, at[0], pc.table[at[1]])
        else:
            logits = self._replay(B, tokens, at)
        for s in seqs:
            pc.lens[s] += 1
        return logits

    def _replay(self, B, tokens, at):
        size = 1 << (B - 1).bit_length()
        g = self.graphs.get(size)
        if g is None:
            g = self.graphs[size] = _StepGraph(self, size)
        g.tokens[:B].copy_(tokens)
        g.pos[:B].copy_(at[0])
        g.pos[B:].fill_(-1)
        g.table[:B].copy_(self.cache.table[at[1]])
        g.graph.replay()
        return g.logits[:B]


class _StepGraph:
    """A decode step of a fixed batch size, captured over static token ids, positions and page tables."""

    def __init__(self, dec, size):
        dev = dec.net.device
        self.tokens = torch.zeros(size, dtype=torch.int64, device=dev)
        self.pos = torch.full((size,), -1, dtype=torch.int64, device=dev)  # captured idle: nothing is appended
        self.table = torch.full((size, dec.cache.table.shape[1]), -1, dtype=torch.int32, device=dev)
        self.graph, self.logits = capture(lambda: dec._forward(self.tokens, self.pos, self.table), dev)
