"""HTTP front end of the B200 engine, with tread's serving contract (tread/server.py:131-237).

    POST /v1/completions   segments in ({prefix, documents[], suffix, tenant, max_tokens,
                           recompute_ratio, policy}), greedy text out, plus the `tread` block of
                           reuse stats (block hits/misses, tokens reused/prefilled, recompute_eff,
                           ttft_ms, total_ms)
    GET  /metrics          request counters and the block store's occupancy and decisions
    GET  /health

Request and response fields, status codes (422 schema, 413 prompt too long, 429 queue full, 503
timed out waiting for the GPU, 401 bad bearer token) and greedy decoding are the reference's,
so a client of the reference server sees the same API. What differs is below the API: prefill is
`tread_b200.Engine.prefill` (host token ids in; one host-to-device copy inside the call) and the
decode steps run the HF model over the `DynamicCache` that prefill hands back, whose layers are
views of the request's assembled cache; with `decoder` (a tread_b200.paged.PagedDecoder) they run
over a paged cache instead, which no token has to copy.

Requests may also carry what the reference has not: repetition_penalty, presence_penalty,
frequency_penalty, logit_bias ({token id: bias}) and allowed_token_ids (a mask over the vocabulary).
They change the logits before the greedy choice (tread_b200.kernels.adjust_logits); left at their
neutral defaults nothing is touched.

The engine is not thread-safe: one lock serialises GPU work; at most `max_queue` requests may be in
flight. Documents are tokenized as untrusted text (control-token text stays plain text); prefix
and suffix are operator-controlled. The tokenizer is shared, so every call to it holds a lock.
"""
import hmac
import threading
import time
from typing import Annotated

import torch
from fastapi import Depends, FastAPI, HTTPException, Request
from pydantic import BaseModel, Field, StringConstraints

from tread_b200 import kernels
from tread_b200.paged import OutOfPages

MAX_SEGMENT_CHARS = 200_000
MAX_DOCUMENTS = 256
# generous characters-per-token bound used to reject huge prompts before tokenizing them
MAX_CHARS_PER_TOKEN = 32


class CompletionRequest(BaseModel):
    prefix: str = Field(min_length=1, max_length=MAX_SEGMENT_CHARS)
    documents: list[Annotated[str, StringConstraints(min_length=1, max_length=MAX_SEGMENT_CHARS)]] = Field(
        default_factory=list, max_length=MAX_DOCUMENTS)
    suffix: str = Field(min_length=1, max_length=MAX_SEGMENT_CHARS)
    tenant: str = Field("", max_length=128)
    max_tokens: int = Field(64, ge=1, le=2048)
    recompute_ratio: float = Field(0.2, ge=0.0, le=1.0)
    policy: str = Field("deviation", pattern="^(deviation|boundary|random)$")
    repetition_penalty: float = Field(1.0, ge=0.01, le=100.0)
    presence_penalty: float = Field(0.0, ge=-100.0, le=100.0)
    frequency_penalty: float = Field(0.0, ge=-100.0, le=100.0)
    logit_bias: dict[int, Annotated[float, Field(ge=-1e4, le=1e4)]] = Field(default_factory=dict, max_length=1024)
    allowed_token_ids: list[int] | None = Field(None, min_length=1, max_length=200_000)


class _Tokenizer:
    """HF tokenizer behind a lock; `untrusted` text is split without special-token parsing."""

    def __init__(self, tok):
        self.tok, self.lock = tok, threading.Lock()

    def encode(self, text, untrusted):
        with self.lock:
            return self.tok(text, add_special_tokens=False, split_special_tokens=untrusted).input_ids

    def decode(self, ids):
        with self.lock:
            return self.tok.decode(ids)


class _Adjust:
    """A request's penalties, biases and mask, applied to its logits step by step; `history` holds the
    prompt's and the answer's token ids on the device."""

    def __init__(self, req, prompt, vocab, device):
        ids = list(req.logit_bias) + (req.allowed_token_ids or [])
        if any(not 0 <= i < vocab for i in ids):
            raise HTTPException(422, f"logit_bias and allowed_token_ids take token ids from 0 to {vocab - 1}")
        self.kw = dict(repetition=req.repetition_penalty, presence=req.presence_penalty,
                       frequency=req.frequency_penalty)
        if req.logit_bias:
            self.kw["bias_ids"] = torch.tensor(list(req.logit_bias), dtype=torch.int64, device=device)
            self.kw["bias"] = torch.tensor(list(req.logit_bias.values()), dtype=torch.float32, device=device)
        if req.allowed_token_ids is not None:
            bits = torch.zeros((vocab + 31) // 32 * 32, dtype=torch.int64)
            bits[torch.tensor(req.allowed_token_ids)] = 1
            words = (bits.view(-1, 32) << torch.arange(32)).sum(1)
            self.kw["allowed"] = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).to(device)
        n = len(prompt)
        self.history = torch.zeros(1, n + req.max_tokens, dtype=torch.int64)
        self.history[0, :n] = torch.tensor(prompt)
        self.history = self.history.to(device)
        self.prompt = torch.tensor([n], device=device)
        self.n = n

    @staticmethod
    def wanted(req):
        return (req.repetition_penalty != 1.0 or req.presence_penalty != 0.0 or req.frequency_penalty != 0.0
                or bool(req.logit_bias) or req.allowed_token_ids is not None)

    def add(self, token):
        self.history[0, self.n] = token
        self.n += 1

    def __call__(self, logits):
        """logits [vocab] -> adjusted fp32 [vocab]."""
        return kernels.adjust_logits(logits[None], tokens=self.history[:, :self.n], prompt_lens=self.prompt,
                                     **self.kw)[0]


def build_app(model, tok, engine, eos_ids, max_context=16384, api_key=None, max_queue=16, queue_timeout=30.0,
              max_seconds=120.0, decoder=None):
    """FastAPI app serving `engine` (a tread_b200.Engine over `model`) with tokenizer `tok`; `decoder`: a
    tread_b200.paged.PagedDecoder over the same model to decode with (default: the HF model)."""
    if decoder is not None and decoder.max_len < max_context:
        raise ValueError(f"decoder: its pages hold sequences of {decoder.max_len} tokens, max_context is {max_context}")

    def auth(request: Request):
        if api_key is not None and not hmac.compare_digest(request.headers.get("authorization", "").encode(),
                                                           f"Bearer {api_key}".encode()):
            raise HTTPException(401, "invalid or missing bearer token", headers={"WWW-Authenticate": "Bearer"})

    app = FastAPI(title="tread_b200", dependencies=[Depends(auth)])
    gpu = threading.Lock()
    slots = threading.BoundedSemaphore(max_queue)
    tk = _Tokenizer(tok)
    eos = set(int(e) for e in eos_ids)
    counters = dict(requests=0, ttft_ms_sum=0.0, tokens_reused=0, tokens_prefilled=0, generated_tokens=0)

    def tokenize(req):
        segs = [(req.prefix, False)] + [(d, True) for d in req.documents] + [(req.suffix, False)]
        if sum(len(t) for t, _ in segs) > max_context * MAX_CHARS_PER_TOKEN:
            raise HTTPException(413, f"prompt exceeds {max_context * MAX_CHARS_PER_TOKEN} characters")
        left, ids = max_context - req.max_tokens, []
        for text, untrusted in segs:
            ids.append(tk.encode(text, untrusted))
            left -= len(ids[-1])
            if left < 0:
                raise HTTPException(413, f"prompt + {req.max_tokens} new tokens exceeds limit {max_context}")
        return ids

    def generate(req, ids):
        host = [torch.tensor(x, dtype=torch.long) for x in ids]
        seq = adjust = None
        if _Adjust.wanted(req):
            adjust = _Adjust(req, [t for seg in ids for t in seg], model.config.vocab_size, model.device)
        pick = lambda logits: int((adjust(logits) if adjust else logits).argmax().item())  # noqa: E731
        with torch.inference_mode():
            t0 = time.perf_counter()
            logits, cache, st = engine.prefill(host[0], host[1:-1], host[-1], ratio=req.recompute_ratio,
                                               policy=req.policy, namespace=req.tenant)
            nxt = pick(logits)
            out, reason = [], "stop"
            dev = logits.device
            try:
                if decoder is not None:
                    seq = decoder.admit(cache, room=req.max_tokens)
                    cache = None
                while nxt not in eos:
                    if len(out) >= req.max_tokens:
                        reason = "length"
                        break
                    if time.perf_counter() - t0 > max_seconds:
                        reason = "time"
                        break
                    out.append(nxt)
                    if adjust:
                        adjust.add(nxt)
                    if decoder is not None:
                        nxt = pick(decoder.step([seq], [nxt])[0])
                    else:
                        o = model(torch.tensor([[nxt]], device=dev), past_key_values=cache, use_cache=True,
                                  logits_to_keep=1)
                        cache, nxt = o.past_key_values, pick(o.logits[0, -1])
                if decoder is not None:
                    decoder.net.check_errors()
            finally:
                if seq is not None:
                    decoder.release(seq)
            total = time.perf_counter() - t0
        counters["requests"] += 1
        counters["ttft_ms_sum"] += st.t["ttft"] * 1e3
        counters["tokens_reused"] += st.tokens_reused
        counters["tokens_prefilled"] += st.tokens_prefilled
        counters["generated_tokens"] += len(out)
        return {
            "text": tk.decode(out),
            "finish_reason": reason,
            "usage": {"prompt_tokens": sum(map(len, ids)), "completion_tokens": len(out)},
            "tread": {"block_hits": st.hits, "block_misses": st.misses, "tokens_reused": st.tokens_reused,
                      "tokens_prefilled": st.tokens_prefilled, "recompute_eff": round(st.recompute_eff, 4),
                      "ttft_ms": round(st.t["ttft"] * 1e3, 2), "total_ms": round(total * 1e3, 2)},
        }

    @app.get("/health")
    def health():
        return {"status": "ok", "model": model.config._name_or_path}

    @app.post("/v1/completions")
    def complete(req: CompletionRequest):
        if not slots.acquire(blocking=False):
            raise HTTPException(429, f"server busy: {max_queue} requests already in flight",
                                headers={"Retry-After": "1"})
        try:
            ids = tokenize(req)
            if not gpu.acquire(timeout=queue_timeout):
                raise HTTPException(503, f"timed out after {queue_timeout}s waiting for the GPU",
                                    headers={"Retry-After": "5"})
            try:
                return generate(req, ids)
            except OutOfPages as e:  # a decoder that others use too
                raise HTTPException(503, f"no room to decode: {e}", headers={"Retry-After": "5"}) from None
            finally:
                gpu.release()
        finally:
            slots.release()

    @app.get("/metrics")
    def metrics():
        s = engine.store.stats
        return {**counters, "ttft_ms_mean": counters["ttft_ms_sum"] / max(1, counters["requests"]),
                "store": {"blocks_gpu": len(engine.store.blocks), "blocks_cpu": len(engine.store.cpu_blocks),
                          "gpu_bytes": s.bytes_used, "cpu_bytes": s.cpu_bytes_used, "hits": s.hits,
                          "misses": s.misses, "cpu_hits": s.cpu_hits, "offloads": s.offloads,
                          "evictions": s.evictions, "cpu_evictions": s.cpu_evictions}}

    return app
