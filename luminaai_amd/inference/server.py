"""HTTP inference server: OpenAI-compatible completions over the
KV-cached GenerationEngine.

The reference ships only a terminal REPL (reference Chat.py:472-937); this
module adds the serving path a production deployment needs: an ASGI app
with /v1/completions, /v1/chat/completions (ChatML via the tokenizer's
conversation encoding), SSE streaming, /health, /v1/models and a
Prometheus /metrics endpoint. The default serving mode is token-level
continuous batching (inference/continuous.py — requests join the running
decode batch between steps; a lone request pays batch-1 compute);
serving="dynamic" keeps request-level batching with the hipGraph
single-stream path for streaming.

Run: python serve.py --checkpoint PATH [--port 8000] [--quantize int8]
"""

from __future__ import annotations

import json
import math
import queue
import threading
import time
from typing import Dict, List, Optional

import torch

from .engine import GenerationConfig, GenerationEngine


def _gen_config(body: Dict) -> GenerationConfig:
    """The request's generation options; raises TypeError or ValueError for
    values that sampling would stumble over."""
    cfg = GenerationConfig.from_mode(body.get("mode", "standard"))
    if "max_tokens" in body:
        cfg.max_new_tokens = int(body["max_tokens"])
    if "temperature" in body:
        cfg.temperature = float(body["temperature"])
    if "top_p" in body:
        cfg.top_p = float(body["top_p"])
    if "top_k" in body:
        cfg.top_k = int(body["top_k"])
    if "repetition_penalty" in body:
        cfg.repetition_penalty = float(body["repetition_penalty"])
    if "stop_token_ids" in body:
        cfg.stop_token_ids = list(body["stop_token_ids"])
        if not all(type(t) is int for t in cfg.stop_token_ids):
            raise ValueError("stop_token_ids must be whole numbers")
    if not (math.isfinite(cfg.temperature) and math.isfinite(cfg.top_p)):
        raise ValueError("temperature and top_p must be finite")
    if 0 < cfg.temperature < 1e-6:          # logits / temperature would overflow
        cfg.temperature = 0.0
    if not 1e-3 <= cfg.repetition_penalty <= 1e3:
        raise ValueError("repetition_penalty must be 0.001 to 1000")
    return cfg


def _paged_options(body: Dict, cfg: GenerationConfig, max_batch: int) -> int:
    """Reads `n` and `logprobs` of a request to a paged server: sets
    cfg.logprobs, returns n."""
    n = 1 if body.get("n") is None else int(body["n"])
    if not 1 <= n <= max_batch:
        raise ValueError(f"n must be 1 to {max_batch}")
    lp = body.get("logprobs")
    if lp is not None and lp is not False:
        # completions: a number; chat: true with top_logprobs beside it
        cfg.logprobs = int(body.get("top_logprobs") or 0 if lp is True else lp)
        if not 0 <= cfg.logprobs <= 64:
            raise ValueError("logprobs must be 0 to 64")
    if body.get("stream") and (n != 1 or cfg.logprobs is not None):
        raise ValueError("a stream takes neither n nor logprobs")
    return n


class _DynamicBatcher:
    """Dynamic request batching: non-streaming requests queue up and are
    decoded together through GenerationEngine.generate_batch (left-padded
    shared KV cache, per-row sampling configs). Requests that arrive while
    a batch is decoding form the next batch — throughput scales with
    concurrency without a latency penalty for the lone request."""

    def __init__(self, engine: GenerationEngine, max_batch: int = 8,
                 window_ms: float = 2.0, lock: Optional[threading.Lock] = None):
        self.engine = engine
        self.lock = lock or threading.Lock()
        self.max_batch = max_batch
        self.window_s = window_ms / 1000.0
        self.q: "queue.Queue" = queue.Queue()
        self.batches_run = 0
        self.rows_seen = 0
        self._thread = threading.Thread(target=self._loop, daemon=True)
        self._thread.start()

    def submit(self, prompt_ids: List[int],
               cfg: GenerationConfig) -> List[int]:
        done = threading.Event()
        slot: Dict = {"ids": prompt_ids, "cfg": cfg, "done": done}
        self.q.put(slot)
        done.wait()
        if "error" in slot:
            raise slot["error"]
        return slot["out"]

    def _loop(self):
        while True:
            batch = [self.q.get()]
            deadline = time.monotonic() + self.window_s
            while len(batch) < self.max_batch:
                remaining = deadline - time.monotonic()
                if remaining <= 0:
                    break
                try:
                    batch.append(self.q.get(timeout=remaining))
                except queue.Empty:
                    break
            try:
                with self.lock:
                    outs = self.engine.generate_batch(
                        [r["ids"] for r in batch], [r["cfg"] for r in batch])
                for r, out in zip(batch, outs):
                    r["out"] = out
            except Exception as e:  # noqa: BLE001
                for r in batch:
                    r["error"] = e
            finally:
                self.batches_run += 1
                self.rows_seen += len(batch)
                for r in batch:
                    r["done"].set()


class _ContinuousWorker:
    """Serving loop over ContinuousBatchingEngine: requests (streaming or
    not) join the running decode batch at token granularity; a lone
    request pays batch-1 compute (active-row compaction). paged: over
    PagedBatchingEngine instead, where a request may ask for several answers
    (forks of its prompt) and for log probabilities."""

    def __init__(self, model, tokenizer, max_batch: int = 8,
                 max_len: int = 2048, paged: bool = False):
        from .continuous import ContinuousBatchingEngine
        from .paged import PagedBatchingEngine
        self.paged = paged
        self.eng = (PagedBatchingEngine if paged else
                    ContinuousBatchingEngine)(model, tokenizer,
                                              max_batch=max_batch,
                                              max_len=max_len)
        self.q: "queue.Queue" = queue.Queue()
        self._thread = threading.Thread(target=self._loop, daemon=True)
        self._thread.start()

    def submit(self, prompt_ids: List[int], cfg: GenerationConfig,
               cb=None) -> List[int]:
        return self.submit_n(prompt_ids, cfg, 1, cb)[0][0]

    def submit_n(self, prompt_ids: List[int], cfg: GenerationConfig,
                 n: int = 1, cb=None) -> List:
        """n answers: (tokens, log probabilities or None) of each."""
        evt = threading.Event()
        item = {"ids": prompt_ids, "cfg": cfg, "cb": cb, "evt": evt, "n": n,
                "out": [None] * n}
        self.q.put(item)
        evt.wait()
        if "err" in item:
            raise item["err"]
        return item["out"]

    @staticmethod
    def _refuse(item: Dict, err: Exception):
        item["err"] = err
        item["evt"].set()

    def _admit(self, items: List[Dict], tracked: Dict):
        """Prefills the requests together (paged) or the only one."""
        try:
            if self.paged:
                slots = self.eng.admit_many([i["ids"] for i in items],
                                            [i["cfg"] for i in items],
                                            [i["cb"] for i in items])
            else:
                slots = [self.eng.admit(i["ids"], i["cfg"], i["cb"])
                         for i in items]
        except Exception as e:  # noqa: BLE001
            if len(items) == 1:
                self._refuse(items[0], e)
            else:                       # one of them is at fault
                for item in items:
                    self._admit([item], tracked)
            return
        for item, b in zip(items, slots):
            tracked[b] = (item, 0)
            try:
                for i in range(1, item["n"]):
                    tracked[self.eng.fork(b)] = (item, i)
            except Exception as e:  # noqa: BLE001
                self._refuse(item, e)

    def _admit_in_order(self, pending: List[Dict], tracked: Dict):
        """paged: all requests from the first on that fit now; what comes later
        does not overtake one that has to wait."""
        for item in list(pending):
            if not self.eng.can_ever_admit(len(item["ids"]), item["n"]):
                pending.remove(item)
                self._refuse(item, RuntimeError(
                    "prompt exceeds the serving context window"))
        while True:
            n = self.eng.admissible([(len(i["ids"]), i["n"])
                                     for i in pending])
            if n == 0:
                return
            items = pending[:n]
            del pending[:n]
            self._admit(items, tracked)

    def _admit_any(self, pending: List[Dict], tracked: Dict):
        """continuous: each request that fits now."""
        for item in list(pending):
            if self.eng.can_admit(len(item["ids"])):
                pending.remove(item)
                self._admit([item], tracked)
            elif self.eng.n_active() == 0:
                pending.remove(item)
                self._refuse(item, RuntimeError(
                    "prompt exceeds the serving context window"))

    def _loop(self):
        # slot -> (request, which of its answers)
        tracked: Dict[int, tuple] = {}
        pending: List[Dict] = []
        while True:
            # drain arrivals; block only when completely idle
            block = not tracked and not pending
            while True:
                try:
                    pending.append(self.q.get(block=block, timeout=None))
                    block = False
                except queue.Empty:
                    break
                if not block:
                    break
            while True:     # opportunistic non-blocking drain
                try:
                    pending.append(self.q.get_nowait())
                except queue.Empty:
                    break
            if self.paged:
                self._admit_in_order(pending, tracked)
            else:
                self._admit_any(pending, tracked)
            if self.eng.n_active():
                try:
                    self.eng.step()
                except Exception as e:  # noqa: BLE001
                    for item, _ in tracked.values():
                        self._refuse(item, e)
                    tracked.clear()
                    for b, s in enumerate(self.eng.slots):
                        if s.active:
                            self.eng._retire(b)
            for b, (item, i) in list(tracked.items()):
                s = self.eng.slots[b]
                if not s.active and s.result is not None:
                    if getattr(s, "error", None) is not None:
                        item["err"] = s.error
                    item["out"][i] = (s.result, getattr(s, "logprobs", None))
                    del tracked[b]
                    if None not in item["out"]:
                        item["evt"].set()


def create_app(model, tokenizer, model_name: str = "luminaai-amd",
               max_batch: int = 8, serving: str = "continuous",
               max_len: int = 2048):
    """Build the ASGI app around an already-loaded model. serving:
    "continuous" (token-level joins, default), "paged" (the same over a paged
    cache, with `n` answers and `logprobs`) or "dynamic" (request-level
    batching with the hipGraph single-stream path for streaming)."""
    from fastapi import FastAPI
    from fastapi.responses import JSONResponse, StreamingResponse

    app = FastAPI(title="LuminaAI-AMD", version="0.1")
    device = next(model.parameters()).device
    engine = GenerationEngine(model, tokenizer, device)
    lock = threading.Lock()
    if serving in ("continuous", "paged"):
        worker = _ContinuousWorker(model, tokenizer, max_batch=max_batch,
                                   max_len=max_len, paged=serving == "paged")
        batcher = None
    else:
        batcher = _DynamicBatcher(engine, max_batch=max_batch, lock=lock)
        worker = None
    started = time.time()
    counters = {"requests": 0, "tokens_out": 0}
    from ..monitoring.prometheus import make_server_metrics
    prom = make_server_metrics()

    def _account(endpoint: str, n_out: int, t0: float):
        counters["requests"] += 1
        counters["tokens_out"] += n_out
        if prom is not None:
            prom["requests"].labels(endpoint=endpoint).inc()
            prom["tokens"].inc(n_out)
            prom["latency"].observe(time.perf_counter() - t0)

    def _decode(prompt_ids: List[int], cfg: GenerationConfig,
                cb=None, endpoint: str = "completions") -> List[int]:
        t0 = time.perf_counter()
        if worker is not None:
            # continuous batching: streaming and non-streaming alike join
            # the running decode batch at token granularity
            out = worker.submit(prompt_ids, cfg, cb=cb)
        elif cb is None:
            # dynamic mode, non-streaming: requests share one batched pass
            out = batcher.submit(prompt_ids, cfg)
        else:
            # dynamic mode, streaming: single-sequence (hipGraph) decode
            with lock:
                out = engine.generate(prompt_ids, cfg, stream_callback=cb)
        _account(endpoint, len(out), t0)
        return out

    def _answers(prompt_ids: List[int], cfg: GenerationConfig, n: int,
                 endpoint: str = "completions") -> List:
        """The request's n answers: (tokens, log probabilities or None)."""
        if serving != "paged":
            return [(_decode(prompt_ids, cfg, endpoint=endpoint), None)]
        t0 = time.perf_counter()
        outs = worker.submit_n(prompt_ids, cfg, n)
        _account(endpoint, sum(len(t) for t, _ in outs), t0)
        return [(t, lp if cfg.logprobs is not None else None)
                for t, lp in outs]

    def _options(body: Dict):
        """(generation options, n, refusal); only paged serving takes more
        than one answer and log probabilities, other modes ignore both."""
        try:
            cfg = _gen_config(body)
            n = _paged_options(body, cfg, max_batch) \
                if serving == "paged" else 1
            return cfg, n, None
        except (TypeError, ValueError, OverflowError) as e:
            return None, 1, JSONResponse({"error": str(e)}, status_code=400)

    def _sse_stream(prompt_ids: List[int], cfg: GenerationConfig,
                    wrap, endpoint: str = "completions") -> StreamingResponse:
        q: "queue.Queue[Optional[int]]" = queue.Queue()

        def run():
            try:
                _decode(prompt_ids, cfg, cb=q.put, endpoint=endpoint)
            finally:
                q.put(None)

        threading.Thread(target=run, daemon=True).start()

        def gen():
            while True:
                tok = q.get()
                if tok is None:
                    break
                piece = tokenizer.decode([tok])
                yield f"data: {json.dumps(wrap(piece))}\n\n"
            yield "data: [DONE]\n\n"

        return StreamingResponse(gen(), media_type="text/event-stream")

    @app.get("/health")
    def health():
        d = {"status": "ok", "device": str(device), "serving": serving,
             "uptime_s": round(time.time() - started, 1), **counters}
        if worker is not None:
            d.update(worker.eng.stats)
        else:
            d.update(batches_run=batcher.batches_run,
                     batched_rows=batcher.rows_seen)
        return d

    @app.get("/metrics")
    def metrics():
        if prom is None:
            return JSONResponse({"error": "prometheus_client not installed"},
                                status_code=501)
        from fastapi.responses import Response
        from prometheus_client import generate_latest
        return Response(generate_latest(prom["registry"]),
                        media_type="text/plain; version=0.0.4")

    @app.get("/v1/models")
    def models():
        return {"object": "list",
                "data": [{"id": model_name, "object": "model"}]}

    @app.post("/v1/completions")
    def completions(body: Dict):
        prompt = body.get("prompt", "")
        cfg, n, refusal = _options(body)
        if refusal is not None:
            return refusal
        ids = tokenizer.encode(prompt)
        if body.get("stream"):
            return _sse_stream(ids, cfg, lambda piece: {
                "object": "text_completion.chunk",
                "choices": [{"text": piece, "index": 0}]})
        outs = _answers(ids, cfg, n)
        n_out = sum(len(t) for t, _ in outs)
        choices = []
        for i, (toks, lps) in enumerate(outs):
            c = {"text": tokenizer.decode(toks), "index": i,
                 "finish_reason": "stop"}
            if lps is not None:
                c["logprobs"] = {
                    "tokens": [tokenizer.decode([e["token"]]) for e in lps],
                    "token_logprobs": [e["logprob"] for e in lps],
                    "top_logprobs": [
                        {tokenizer.decode([t]): p for t, p in e["top"]}
                        for e in lps]}
            choices.append(c)
        return JSONResponse({
            "object": "text_completion",
            "model": model_name,
            "choices": choices,
            "usage": {"prompt_tokens": len(ids),
                      "completion_tokens": n_out,
                      "total_tokens": len(ids) + n_out},
        })

    @app.post("/v1/chat/completions")
    def chat_completions(body: Dict):
        messages = body.get("messages", [])
        cfg, n, refusal = _options(body)
        if refusal is not None:
            return refusal
        ids: List[int] = []
        for m in messages:
            ids.extend(tokenizer.encode_message(m.get("role", "user"),
                                                m.get("content", "")))
        # open the assistant turn so decoding continues it
        ids.extend(tokenizer.encode_message("assistant", "")[:-1])
        if body.get("stream"):
            return _sse_stream(ids, cfg, lambda piece: {
                "object": "chat.completion.chunk",
                "choices": [{"delta": {"content": piece}, "index": 0}]},
                endpoint="chat")
        outs = _answers(ids, cfg, n, endpoint="chat")
        n_out = sum(len(t) for t, _ in outs)
        choices = []
        for i, (toks, lps) in enumerate(outs):
            c = {"message": {"role": "assistant",
                             "content": tokenizer.decode(toks)},
                 "index": i, "finish_reason": "stop"}
            if lps is not None:
                c["logprobs"] = {"content": [
                    {"token": tokenizer.decode([e["token"]]),
                     "logprob": e["logprob"],
                     "top_logprobs": [{"token": tokenizer.decode([t]),
                                       "logprob": p} for t, p in e["top"]]}
                    for e in lps]}
            choices.append(c)
        return JSONResponse({
            "object": "chat.completion",
            "model": model_name,
            "choices": choices,
            "usage": {"prompt_tokens": len(ids),
                      "completion_tokens": n_out,
                      "total_tokens": len(ids) + n_out},
        })

    return app


def main(argv=None):
    import argparse

    from ..data.tokenizer import ConversationTokenizer
    from ..models import DeepSeekTransformer
    from .loader import (find_latest_checkpoint, infer_config_from_state_dict,
                         load_checkpoint_smart)

    ap = argparse.ArgumentParser(description="LuminaAI-AMD inference server")
    ap.add_argument("--checkpoint", default=None)
    ap.add_argument("--host", default="127.0.0.1")
    ap.add_argument("--port", type=int, default=8000)
    ap.add_argument("--device", default=None)
    ap.add_argument("--quantize", default=None,
                    choices=["int8", "int4", "fp8"])
    ap.add_argument("--max-batch", type=int, default=8,
                    help="continuous-batching slot count")
    ap.add_argument("--max-len", type=int, default=2048,
                    help="serving context window (KV cache columns)")
    ap.add_argument("--serving", default="continuous",
                    choices=["continuous", "paged", "dynamic"])
    args = ap.parse_args(argv)

    device = torch.device(args.device) if args.device else (
        torch.device("cuda") if torch.cuda.is_available()
        else torch.device("cpu"))
    path = args.checkpoint or find_latest_checkpoint()
    if path is None:
        raise SystemExit("no checkpoint found; pass --checkpoint")
    payload = load_checkpoint_smart(path)
    sd = payload["model_state_dict"]
    cfg = infer_config_from_state_dict(sd)
    model = DeepSeekTransformer(cfg)
    model.load_state_dict(sd, strict=False)
    model = model.to(device).eval()
    if device.type == "cuda":
        model = model.to(torch.bfloat16)
    if args.quantize:
        from ..ops.quant import quantize_model
        n = quantize_model(model, mode=args.quantize)
        print(f"quantized {n} Linear layers to {args.quantize}")

    app = create_app(model, ConversationTokenizer(),
                     max_batch=args.max_batch, serving=args.serving,
                     max_len=args.max_len)
    import uvicorn
    uvicorn.run(app, host=args.host, port=args.port, log_level="info")


if __name__ == "__main__":
    main()
