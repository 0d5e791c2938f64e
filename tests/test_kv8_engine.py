"""The 8-bit cache in the engine and around it: status words, models, generated tokens."""
from types import SimpleNamespace as NS

import pytest
import torch

gpu = pytest.mark.gpu


def test_the_step_reads_the_status_word_of_its_own_device(monkeypatch):
    """A process whose first kernels ran on another device: waits that give up in this device's attention are reported, too."""
    from vllm_kunlun_b200.engine.runner import ModelRunner
    from vllm_kunlun_b200.ops import _ext
    words = {0: NS(device=torch.device("cuda:0")), 1: NS(device=torch.device("cuda:1"))}
    monkeypatch.setattr(_ext, "available", lambda: True)
    monkeypatch.setattr(_ext, "C", lambda: NS(gemm_status_tensor=lambda device=None: words.get(0 if device is None else device)))

    def read(device):
        runner = NS(pstate=NS(tp_comm=None), device=torch.device(device), _status_cache=None)
        return [w for _, w in ModelRunner._status_words(runner)]
    assert read("cuda:0") == [words[0]]
    assert read("cuda:1") == [words[0], words[1]]
    assert read("cuda:2") == [words[0]]            # nothing of the kind has run there


@gpu
def test_status_words_by_device():
    from test_kv8 import attend, batch
    from vllm_kunlun_b200.ops import _ext, gemm_cuda
    attend(batch([1], [40], 4, 2, 128, 64, torch.bfloat16, "cuda"))
    word = _ext.C().gemm_status_tensor()
    here = _ext.C().gemm_status_tensor(torch.cuda.current_device())
    assert here is not None and here.device.index == torch.cuda.current_device()
    assert _ext.C().gemm_status_tensor(torch.cuda.device_count()) is None
    assert word is not None and int(here) == 0
    here.fill_(905)
    try:
        with pytest.raises(RuntimeError):
            gemm_cuda.check_status()
    finally:
        here.zero_()
    gemm_cuda.check_status()


# ----------------------------------------------------------------------------- models

def model(name, head_dim=32, dtype="float32", hidden=64, heads=(2, 1), inter=128, expert=64):
    from vllm_kunlun_b200.config import gpt_oss_20b, llama_3_1_8b, qwen2_0_5b, qwen3_30b_a3b, qwen3_8b, qwen3_next_80b_a3b, tiny
    kw = dict(vocab_size=128, hidden_size=hidden, num_heads=heads[0], num_kv_heads=heads[1], head_dim=head_dim, intermediate_size=inter,
              max_position=512, dtype=dtype)
    moe = dict(num_experts=4, num_experts_per_tok=2, moe_intermediate_size=expert)
    if name == "dense":
        return tiny(llama_3_1_8b(), num_layers=2, **kw)
    if name == "normed":
        return tiny(qwen3_8b(), num_layers=2, **kw)
    if name == "experts":
        return tiny(qwen3_30b_a3b(fp8=False), num_layers=2, **kw, **moe)
    if name == "sinks and windows":
        return tiny(gpt_oss_20b(), num_layers=2, **kw, **moe, sliding_window=24)
    if name == "narrow values":
        cfg = tiny(qwen3_30b_a3b(fp8=False), num_layers=2, **kw, **moe, v_head_dim=head_dim // 2)
        cfg.architecture = "MiMoV2FlashForCausalLM"
        return cfg
    if name == "shared layers":
        cfg = tiny(llama_3_1_8b(), num_layers=6, **kw)
        cfg.architecture, cfg.hidden_act = "Gemma4ForCausalLM", "gelu_tanh"
        cfg.gemma_norm = cfg.qk_norm = cfg.tie_word_embeddings = True
        cfg.sliding_window, cfg.sliding_window_pattern = 20, 3
        cfg.num_kv_shared_layers, cfg.final_logit_softcapping, cfg.attn_scale = 2, 30.0, 1.0
        return cfg
    if name == "hybrid":
        return tiny(qwen3_next_80b_a3b(), num_layers=4, **kw, **moe, rotary_dim=8, gdn_num_k_heads=2, gdn_num_v_heads=4,
                    gdn_head_k_dim=16, gdn_head_v_dim=16)
    assert name == "images"
    cfg = tiny(qwen2_0_5b(), num_layers=2, **kw)
    cfg.architecture = "Qwen2_5_VLForConditionalGeneration"
    cfg.vision = dict(depth=2, hidden=32, heads=2, patch=2, temporal_patch=1, merge=2, intermediate=64, in_channels=3, norm="rmsnorm",
                      gated_mlp=True, image_token_id=127, text_architecture="Qwen2ForCausalLM")
    cfg.mrope_section = (4, 6, 6)
    return cfg


MODELS = ["dense", "normed", "experts", "sinks and windows", "narrow values", "shared layers", "hybrid", "images"]


def generate(cfg, kind, device="cpu", weights=None, steps=6, **kw):
    """Tokens of three prompts in chunks, the logits of every step, and the engine."""
    from vllm_kunlun_b200 import LLM, SamplingParams
    llm = LLM(cfg, device=device, block_size=16, max_model_len=256, max_num_seqs=4, num_gpu_blocks=64, max_num_batched_tokens=48, seed=5,
              kv_cache_dtype=kind, **kw)
    m = llm.engine.runner.model
    if weights is not None:
        with torch.inference_mode():
            m.load_state_dict(weights)
    logits, compute = [], m.compute_logits

    def recorded(hidden):
        out = compute(hidden)
        if out.numel():                        # a step of chunks alone has none
            logits.append(out.float().cpu())
        return out
    if device == "cpu" or kw.get("enforce_eager"):
        m.compute_logits = recorded
    prompts = [[3 + (7 * i + j) % 119 for i in range(n)] for j, n in enumerate((70, 3, 33))]
    extra = {}
    if cfg.architecture.startswith("Qwen2_5_VL"):
        px = torch.randn(32, 12, generator=torch.Generator().manual_seed(0))
        prompts[1] = [5, 6, 7] + [127] * 8 + [9, 10]
        extra = dict(multi_modal_data=[None, {"pixel_values": px, "image_grid_thw": [(1, 8, 4)]}, None])
    out = [list(o.token_ids) for o in llm.generate(prompts, SamplingParams(max_tokens=steps, temperature=0.0, ignore_eos=True), **extra)]
    return out, logits, llm


@pytest.mark.parametrize("name", MODELS)
def test_models_read_what_they_wrote(monkeypatch, name):
    """fp32 models on an 8-bit cache against the same models on a cache of their own type that holds what the 8-bit one stands for."""
    from vllm_kunlun_b200.ops.reference import attention as ra
    got, logits, llm = generate(model(name), "fp8_e4m3")
    paged = [t for c in llm.engine.runner.kv_caches.values() for t in (c if isinstance(c, tuple) else (c,)) if t.dim() == 5]
    assert paged and all(t.dtype == torch.uint8 for t in paged)
    plain = generate(model(name), "auto")[1]
    put = ra.reshape_and_cache

    def rounded(k, v, cache, slots):
        codes, scales = ra.kv8_rows(k, v)
        x = codes.float() * scales[..., None]
        put(x[:, 0], x[:, 1], cache, slots)
    monkeypatch.setattr(ra, "reshape_and_cache", rounded)
    want, exact, _ = generate(model(name), "auto")
    assert got == want and len(logits) == len(exact)
    # some hundred fp32 roundings of 2^-24 in a row, relative to the largest logit
    for a, b in zip(logits, exact):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()
    # ... which is well below what 8 bits change
    assert any((a - b).abs().max() > 1e-3 * b.abs().max() for a, b in zip(plain, exact) if a.shape == b.shape)


def test_verification_from_an_8_bit_cache():
    """Drafts of the prompt's own n-grams: the tokens are those of plain decoding from the same cache."""
    cfg = model("normed")
    want = generate(cfg, "fp8_e4m3", steps=20)[0]
    got, _, llm = generate(cfg, "fp8_e4m3", steps=20, speculative_config={"method": "ngram", "num_speculative_tokens": 3})
    assert got == want and llm.engine.stats["spec_proposed"] > 0


def test_draft_layers_keep_their_own_type():
    """EAGLE's layers stay in the model's type beside the target's 8-bit cache, and do not change its greedy tokens."""
    from vllm_kunlun_b200.config import llama_3_1_8b, tiny
    cfg = tiny(llama_3_1_8b(), num_layers=4, vocab_size=128, hidden_size=64, num_heads=2, num_kv_heads=1, head_dim=32,
               intermediate_size=128, max_position=512, dtype="float32")
    want = generate(cfg, "fp8_e4m3", steps=10)[0]
    got, _, llm = generate(cfg, "fp8_e4m3", steps=10, speculative_config={"method": "eagle", "num_speculative_tokens": 1})
    assert got == want
    kinds = [llm.engine.runner.kv_caches[i].dtype for i in sorted(llm.engine.runner.kv_caches)]
    assert kinds == [torch.uint8] * 4 + [torch.float32]


def test_models_of_listed_layers_refuse():
    from vllm_kunlun_b200.models.layer_list import LayerListForCausalLM
    with pytest.raises(ValueError, match="fp8_e4m3"):
        LayerListForCausalLM.kv_cache_spec(NS(kv_cache_dtype="fp8_e4m3"), 16)


@gpu
@pytest.mark.parametrize("name", ["dense", "normed", "shared layers"])          # experts need 16 bits there
def test_models_on_the_gpu(name):
    """fp32: the tokens of the same weights on the CPU; chunked prompts, mixed steps, decode steps from captured graphs."""
    cfg = model(name)
    want, _, cpu = generate(cfg, "fp8_e4m3", steps=12)
    got = generate(model(name), "fp8_e4m3", "cuda", cpu.engine.runner.model.state_dict(), steps=12)[0]
    assert got == want


@gpu
@pytest.mark.parametrize("name", ["dense", "normed", "experts"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_bf16_models_on_the_gpu(monkeypatch, name, head_dim):
    """The tensor-core kernels in the engine: logits of the first steps (one token of every prompt, then decode steps while the tokens
    agree) against the same weights in fp32 on the CPU.

    A layer has some fifteen roundings to bf16 in a row, two layers and the head: 31 * 2^-8 if they all added up, 2^-8 * 31 ** 0.5 < 2^-5 as
    independent errors of a norm; codes that fall to the other side of a rounding change a key or a value by 2^-3 of an element, one in
    sixteen of them or so: 2^-5.  Together 2^-4."""
    from vllm_kunlun_b200.ops.reference import attention as ra
    size = dict(hidden=512, heads=(8, 2), inter=1024, expert=256)
    toks, got, gpu_llm = generate(model(name, head_dim, "bfloat16", **size), "fp8_e4m3", "cuda", enforce_eager=True)
    weights = {k: v.float().cpu() if v.is_floating_point() else v.cpu() for k, v in gpu_llm.engine.runner.model.state_dict().items()}
    want_toks, want, _ = generate(model(name, head_dim, **size), "fp8_e4m3", weights=weights)
    same = next((i for i in range(6) if any(a[i] != b[i] for a, b in zip(toks, want_toks))), 6)
    assert len(got) == len(want)
    # the logits of step i have seen the tokens in front of i
    off = [float(((a - b).norm(dim=-1) / b.norm(dim=-1)).max()) for a, b in list(zip(got, want))[:same + 1 if same < 6 else None]]
    assert max(off) <= 2.0 ** -4, (off, same)
    # a cache that held nothing would show
    monkeypatch.setattr(ra, "gather_kv_cache", lambda cache, slots, dtype: [torch.zeros(len(slots), cache.shape[2], cache.shape[4] - 4,
                                                                                        dtype=dtype)] * 2)
    empty = generate(model(name, head_dim, **size), "fp8_e4m3", weights=weights)[1]
    assert float(((empty[0] - want[0]).norm(dim=-1) / want[0].norm(dim=-1)).max()) > 2.0 ** -2


@gpu
def test_experts_of_other_types_are_refused():
    """Rows of 32 bits: an error, not a wait that gives up."""
    from vllm_kunlun_b200.ops import _ext
    x, w = torch.zeros(4, 64, device="cuda"), torch.zeros(2, 64, 64, device="cuda")
    lod = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    bias = torch.zeros(2, 64, device="cuda")
    for out in (torch.zeros(4, 64, device="cuda"), torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")):
        with pytest.raises(RuntimeError, match="8 or 16 bits"):
            _ext.C().grouped_gemm(out, x, w, lod, bias, None, None, 0, 0)
