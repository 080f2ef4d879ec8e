"""Text generation over the paged cache (reference: stream_tokens / generate_samples_from_prompt,
megatron/text_generation_utils.py:187-402), for a `harness.MagmaStack`.

One step: the image prefix and the prompts of all sequences enter as packed rows; every further step brings one token a
sequence.  The token step reads everything that changes from device memory (tokens, lengths, random numbers), so it is captured
into a HIP graph once and replayed: a 24-layer step is some 200 launches of a few microseconds each.
"""
import torch

from . import mpu, ops
from .kv_cache import PagedKVCache, PagedPast, PagedStep


def _layers(stack, x, cache, step, max_positions):
    for layer, kv in zip(stack.layers, cache.layers):
        x = layer(x, None, layer_past=PagedPast(kv, step, max_positions))
    return x


def _head(stack, rows, vocab_size):
    """Logits [n, vocab_size] of rows [n, 1, h]: final LayerNorm and LM head; the padded vocabulary's tail is cut off."""
    logits, _ = stack.final_linear(stack.final_norm(rows))
    return logits.view(rows.size(0), -1)[:, :vocab_size]


def make_cache(stack, sequences, tokens, page_size=16):
    """A cache for `sequences` sequences of up to `tokens` tokens (image prefix included) of this stack."""
    args = stack.args
    heads = mpu.divide(args.num_attention_heads, mpu.get_model_parallel_world_size())
    w = stack.word_embeddings.weight
    return PagedKVCache(len(stack.layers), heads, args.hidden_size // args.num_attention_heads, sequences * -(-tokens // page_size),
                        page_size=page_size, dtype=w.dtype, device=w.device)


@torch.no_grad()
def generate(stack, prompts, enc_out=None, maximum_tokens=64, eos_token_id=None, temperature=0.0, top_k=0, top_p=0.0, min_p=0.0,
             generator=None, vocab_size=None, cache=None, page_size=16, graph=True):
    """Continue each prompt by up to maximum_tokens tokens.  prompts: list of int64 token tensors or lists (an empty one needs an
    image); enc_out [b, P, enc_dim] the pooled encoder outputs, or None; temperature / top_k / top_p as the reference's arguments
    (0: the most likely token / off / off) and min_p, numbers or [b] tensors (ops.sample_tokens); generator: torch generator on
    the stack's device for the random numbers; vocab_size: the tokens to draw from (default: the padded vocabulary); cache: a
    PagedKVCache of the stack's layers with free pages for all of it (default: one is made).  graph=False: launch every token step
    eagerly.  Returns a list of int64 tensors on the CPU, each up to and with eos_token_id, or with -1 where the logits held a NaN
    (the sequence ends there).  The stack must be in eval mode."""
    if stack.training:
        raise RuntimeError("generate: put the stack in eval mode (dropout has no place here)")
    if mpu.get_model_parallel_world_size() > 1:
        raise NotImplementedError("generate: the sampled distribution is not vocabulary-parallel (tensor-parallel size 1 only)")
    w = stack.word_embeddings.weight
    dev, h = w.device, w.size(1)
    prompts = [torch.as_tensor(p, dtype=torch.int64).reshape(-1).cpu() for p in prompts]
    b = len(prompts)
    if b == 0 or maximum_tokens < 1:
        return [torch.empty(0, dtype=torch.int64) for _ in prompts]
    prefix = None
    if enc_out is not None:
        if stack.image_prefix is None or enc_out.size(0) != b:
            raise RuntimeError(f"generate: enc_out must be [{b}, P, enc_dim] and the stack must have an image prefix")
        prefix = stack.image_prefix(enc_out).view(b, -1, h)
    p_len = prefix.size(1) if prefix is not None else 0
    lens = [p_len + len(p) for p in prompts]
    if min(lens) < 1:
        raise RuntimeError("generate: an empty prompt without an image has nothing to continue")
    total = [n + maximum_tokens - 1 for n in lens]  # the last token drawn enters no cache
    if vocab_size is not None and not 0 < vocab_size <= w.size(0):
        raise RuntimeError(f"generate: vocab_size {vocab_size} is not in (0, {w.size(0)}]")
    if cache is None:
        cache = make_cache(stack, b, max(total), page_size)
    elif len(cache.layers) != len(stack.layers):
        raise RuntimeError(f"generate: a cache of {len(cache.layers)} layers for a stack of {len(stack.layers)}")
    seqs = []
    try:
        for n in total:
            seqs.append(cache.add(n))
        with torch.cuda.device(dev):  # the captured step's stream is the current device's
            return _generate(stack, prompts, prefix, p_len, lens, max(total), cache, seqs, maximum_tokens, eos_token_id,
                             dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p), generator,
                             vocab_size or w.size(0), graph)
    finally:
        for s in seqs:
            cache.release(s)


def _generate(stack, prompts, prefix, p_len, lens, positions, cache, seqs, maximum_tokens, eos, sampling, generator, vocab_size, graph):
    w = stack.word_embeddings.weight
    dev, h, b = w.device, w.size(1), len(prompts)
    # the prompt step: each sequence's prefix rows, then its tokens, packed
    step = cache.step(seqs, lens, lens)
    tokens = torch.cat([torch.cat((torch.zeros(p_len, dtype=torch.int64), p)) for p in prompts]).to(dev)
    x = ops.embed_prefix(w, tokens.view(1, -1))
    if prefix is not None:
        rows = torch.cat([step.cu_new[:-1].long() + i for i in range(p_len)]).view(p_len, b).t().reshape(-1)
        x.view(-1, h).index_copy_(0, rows, prefix.reshape(-1, h))
    x = _layers(stack, x, cache, step, positions)
    last = x.view(-1, h).index_select(0, step.cu_new[1:].long() - 1).view(b, 1, h)
    u = torch.rand(maximum_tokens, b, generator=generator, device=dev)
    out = torch.empty(maximum_tokens, b, dtype=torch.int64, device=dev)
    token = ops.sample_tokens(_head(stack, last, vocab_size), u[0], **sampling)
    out[0] = token
    if maximum_tokens == 1:
        return _trim(out, eos)

    # the token step: every array it reads is rewritten in place between the steps
    kv_lens = torch.tensor([n + 1 for n in lens], dtype=torch.int32).to(dev)
    one = PagedStep(step.block_table, torch.arange(b + 1, dtype=torch.int32).to(dev), kv_lens, max_new=1, max_kv=positions)
    draw = u[1].clone()

    def token_step():
        y = ops.embed_prefix(w, token.view(1, b))
        y = _layers(stack, y, cache, one, positions)
        ops.sample_tokens(_head(stack, y, vocab_size), draw, out=token, **sampling)

    replay = None
    for t in range(1, maximum_tokens):
        if t > 1:
            kv_lens.add_(1)
            draw.copy_(u[t])
        if replay is not None:
            replay.replay()
        else:
            token_step()
            if graph and t == 1 and maximum_tokens > 3:  # the eager step above was the warm-up; capturing runs nothing
                replay = torch.cuda.CUDAGraph()
                with torch.cuda.graph(replay):
                    token_step()
        out[t] = token
        if t % 16 == 0 and eos is not None and bool(_ends(out[:t + 1], eos).any(dim=0).all()):
            out = out[:t + 1]
            break
    return _trim(out, eos)


def _ends(tokens, eos):
    return tokens == -1 if eos is None else (tokens == eos) | (tokens == -1)


def _trim(out, eos):
    rows = out.t().cpu()
    return [r[:int(e.nonzero()[0]) + 1] if bool(e.any()) else r for r, e in zip(rows, _ends(rows, eos))]
