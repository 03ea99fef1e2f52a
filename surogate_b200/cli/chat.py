"""``surogate chat <model dir> [--adapter dir]``: a minimal interactive / one-shot generation loop for checking a trained model.

Answers come from ``Trainer.generate``: a paged key/value cache where the model's layers allow one, else the whole prefix for every token.

Parity: scripts/chat.py.
"""
from __future__ import annotations

import argparse
import sys
from typing import List, Optional


def generate(trainer, tokenizer, prompt_ids: List[int], max_new_tokens: int = 64, temperature: float = 0.0, seed: int = 0, eos_id: Optional[int] = None, top_k: int = 0,
             top_p: float = 1.0, min_p: float = 0.0) -> List[int]:
    eos = tokenizer.eos_token_id if eos_id is None and tokenizer is not None else eos_id
    return trainer.generate([prompt_ids], max_new_tokens=max(0, max_new_tokens), temperature=temperature if temperature > 0 else 0.0, top_k=top_k, top_p=top_p, min_p=min_p, seed=seed, eos_id=eos)[0][0].tokens


def main(argv, command: str = "chat") -> int:
    p = argparse.ArgumentParser(prog="surogate chat")
    p.add_argument("model")
    p.add_argument("--adapter", default=None)
    p.add_argument("--prompt", default=None, help="answer this prompt and exit (otherwise read prompts from stdin)")
    p.add_argument("--max-new-tokens", type=int, default=128)
    p.add_argument("--temperature", type=float, default=0.0)
    p.add_argument("--top-k", type=int, default=0, help="draw from the K likeliest tokens only (0: all)")
    p.add_argument("--top-p", type=float, default=1.0, help="draw from the likeliest tokens that make up this share of the probability")
    p.add_argument("--min-p", type=float, default=0.0, help="leave out tokens less likely than this share of the likeliest one")
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args(argv)
    import torch

    from ..data.tokenizer import Tokenizer
    from ..dsl.compiler import load_hf_config
    from ..runtime.trainer import Trainer, TrainerConfig

    tok = Tokenizer.from_pretrained(a.model)
    cfg = load_hf_config(a.model)
    lora = None
    if a.adapter:
        import json
        import os

        with open(os.path.join(a.adapter, "adapter_config.json")) as f:
            ac = json.load(f)
        lora = dict(rank=ac["r"], alpha=ac["lora_alpha"], dropout=0.0, dtype="fp32", targets=ac["target_modules"], rslora=ac.get("use_rslora", False), train_router=False)
    tr = Trainer(TrainerConfig(model=cfg, batch_size=1, seq_len=128, zero_level=0, lora=lora), device=torch.device("cuda" if torch.cuda.is_available() else "cpu"))
    tr.import_weights(a.model)
    if a.adapter:
        tr.lora.load_peft(a.adapter)

    def answer(text: str) -> str:
        ids = tok.apply_chat_template_and_encode([{"role": "user", "content": text}], add_generation_prompt=True)
        return tok.decode(generate(tr, tok, ids, a.max_new_tokens, a.temperature, a.seed, top_k=a.top_k, top_p=a.top_p, min_p=a.min_p), skip_special_tokens=True)

    if a.prompt is not None:
        print(answer(a.prompt))
        return 0
    for line in sys.stdin:
        if line.strip():
            print(answer(line.strip()), flush=True)
    return 0
