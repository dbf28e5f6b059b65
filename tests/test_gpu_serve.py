"""The serving loop over paged caches (PagedLlama) against the same blocks run over whole
sequences (dispatched_forward, flash attention): logits of prompts that enter in chunks, of
single tokens, and of several sequences at once.

Both paths compute the same network; what differs is roundings: the flash path rounds scores and
each rotation product to fp16, this one only rotated keys and (8-bit tiers) the cached values.
An fp16 chain of 3 layers is within 2 % in the norm; INT8 pages add steps of 1 / 254 of a block's
largest value (about 1 % of a typical one), FP8 pages 2^-4 at most (about 2.5 % rms): 5 % and 10 %.
"""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

BOUND = {0: 0.05, 1: 0.10, 2: 0.02}


@pytest.fixture(scope="module")
def model(cuda):
    from transformers import LlamaConfig
    from transformers.models.llama.modeling_llama import LlamaForCausalLM

    torch.manual_seed(3)
    cfg = LlamaConfig(hidden_size=512, num_hidden_layers=3, num_attention_heads=8, num_key_value_heads=2,
                      intermediate_size=1024, vocab_size=512, rms_norm_eps=1e-5, rope_theta=10000.0,
                      max_position_embeddings=4096, attn_implementation="eager", initializer_range=0.04)
    return LlamaForCausalLM(cfg).cuda().half().eval()


def _blocks(pkg, model):
    # thresholds below every entropy: all rows in the FP16 tier, so that a routing decision near a
    # threshold cannot differ between the two paths
    return pkg.build_dispatched_llama(model, -2.0, -1.0, routing="token", attention="flash")


@pytest.mark.parametrize("tier", [0, 1, 2])
@torch.no_grad()
def test_logits_match_the_whole_sequence(pkg, cuda, model, tier):
    blocks, d = _blocks(pkg, model)
    serve = pkg.PagedLlama(model, blocks, d, max_seqs=3, num_pages=60, page_size=16, tier=pkg.PrecisionTier(tier))
    g = torch.Generator().manual_seed(1)
    lengths = [150, 37, 64]
    ids = [torch.randint(0, 512, (n,), generator=g).tolist() for n in lengths]
    want = [pkg.llama.dispatched_forward(model, blocks, d, torch.tensor([x], device=cuda))[0].float() for x in ids]
    got = [[] for _ in ids]
    at = [0, 0, 0]
    turn = 0
    while any(a < n for a, n in zip(at, lengths)):
        sizes = [(70, 1, 16), (1, 20, 1), (60, 1, 33)][turn % 3]
        take = [min(m, n - a) for m, n, a in zip(sizes, lengths, at)]
        act = [s for s in range(3) if take[s] > 0]
        logits = serve.forward([ids[s][at[s]:at[s] + take[s]] for s in act], act).float()
        row = 0
        for s in act:
            got[s].append(logits[row:row + take[s]])
            row += take[s]
            at[s] += take[s]
        turn += 1
    torch.cuda.synchronize()
    assert pkg._lib.device_check() == 0
    for a, b in zip(got, want):
        a = torch.cat(a)
        assert ((a - b).norm() / b.norm()).item() < BOUND[tier]


@torch.no_grad()
def test_generate_does_not_depend_on_company_or_chunks(pkg, cuda, model):
    """Greedy tokens of prompts served together, alone and in small chunks."""
    blocks, d = _blocks(pkg, model)
    serve = pkg.PagedLlama(model, blocks, d, max_seqs=4, num_pages=40, page_size=16, tier=pkg.PrecisionTier.FP16)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (50, 1, 17)]
    together = serve.generate(prompts, 5)
    assert [len(x) for x in together] == [5, 5, 5]
    assert serve.caches[0].free_pages == 40 and serve.caches[-1].lengths == [0] * 4
    # the first token follows from the prompt alone, whatever the sizes of the steps: compare by
    # logits, as near ties may fall either way
    for p, t in zip(prompts, together):
        logits = serve.forward([p], [0])[-1].float()
        assert logits.max() - logits[t[0]] <= 0.02 * logits.norm()
        serve.release(0)
    assert len(serve.generate(prompts, 3, chunk=7)[0]) == 3
    with pytest.raises(RuntimeError, match="none of them empty"):
        serve.generate([[]], 1)
    with pytest.raises(RuntimeError, match="more than 40 pages"):
        serve.generate([prompts[1], prompts[0] * 20], 1)
    assert serve.caches[0].free_pages == 40  # nothing is left behind
    serve.forward([prompts[2]], [1])
    with pytest.raises(RuntimeError, match="in use"):
        serve.generate(prompts, 1)
    serve.release(1)
    with pytest.raises(RuntimeError, match="routing='token'"):
        pkg.PagedLlama(model, pkg.build_dispatched_llama(model, 0.4, 1.7)[0], d, 1, 8)
