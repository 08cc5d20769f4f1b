"""The 4-bit cache pool and the e4m3 projections on the framework's own paths: the
pool's prefills, commits and views, one packed wave through the target stack, the
attention function of transformers models, and whole decodes.

* Pool contents are exact: the packing of tests/mx4_cases.py, read back as bf16.
* A wave over a 4-bit pool is compared with an fp32 restatement on the CPU whose
  prefixes are the values that the pool holds.  What is left are the roundings that
  the bf16 stack over a bf16 pool of the same values makes too, so its error is
  bounded by that one's, with the allowance (25 %) that the bf16 stack itself has
  against transformers.
* With e4m3 projections the stack's stages are compared, bit for bit, with the public
  operators called one by one, and the outcome with the bf16 stack over the same
  (unpacked) weights: each of a layer's four products sees its rows rounded by at most
  2^-4 of a value (e4m3's half step), which moves a product by less than 2^-4 of its
  norm as long as the weights treat the error no better than the row itself.
"""
import copy
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from specgrove_amd import workloads as W
from tests import mx4_cases
from tests import test_gpu_decode as decode_cases
from tests import test_gpu_target_stack as stack_cases

pytestmark = pytest.mark.gpu


class _Layer:
    def __init__(self, keys, values):
        self.keys, self.values = keys, values


class _Cache:
    def __init__(self, layers):
        self.layers = layers

    def get_seq_length(self):
        return int(self.layers[0].keys.shape[-2])


def _held(x):
    """The values a 4-bit cache holds of bf16 rows x, in bf16 (exact)."""
    x = x.cpu()
    return mx4_cases.values(*mx4_cases.pack(x)).to(torch.bfloat16) if x.numel() else x


def _source(device, length, layers, hkv, dim, layout, seed):
    g = torch.Generator().manual_seed(seed)

    def rows():
        x = torch.randn((1, hkv, length, dim), generator=g).to(torch.bfloat16).to(device)
        if layout == "tokens":     # [L, Hkv, D] memory, as projections write it
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "sliced":     # rows of a longer buffer
            wide = torch.zeros((1, hkv, length + 5, dim), dtype=x.dtype, device=device)
            wide[:, :, 2:2 + length] = x
            return wide[:, :, 2:2 + length]
        if layout == "odd":        # neither aligned rows nor a contiguous last dimension
            return x.transpose(2, 3).contiguous().transpose(2, 3)
        return x
    return _Cache([_Layer(rows(), rows()) for _ in range(layers)])


@pytest.mark.parametrize("layout", ["plain", "tokens", "sliced", "odd"])
@pytest.mark.parametrize("hkv,dim", [(2, 64), (1, 128), (8, 128)])
def test_prefills_are_packed_into_their_slots(device, hkv, dim, layout):
    from specgrove_amd.cache import Mx4RequestCachePool
    lengths = [5, 0, 33, 1, 70]
    caches = [_source(device, L, 3, hkv, dim, layout, 10 * i + dim)
              for i, L in enumerate(lengths)]
    pool = Mx4RequestCachePool(caches, 70)
    pool.check_status()
    assert pool.lengths == lengths and pool.num_layers == 3
    for view, cache in zip(pool.caches, caches):
        assert view.get_seq_length() == cache.get_seq_length()
        for layer, source in zip(view.layers, cache.layers):
            for got, want in ((layer.keys, source.keys), (layer.values, source.values)):
                assert got.dtype == torch.bfloat16
                assert torch.equal(got.cpu(), _held(want))


def test_pool_refusals(device):
    from specgrove_amd.cache import Mx4RequestCachePool
    good = _source(device, 4, 2, 2, 64, "plain", 0)
    with pytest.raises(ValueError, match="capacity is below"):
        Mx4RequestCachePool([good], 3)
    with pytest.raises(ValueError, match="head_dim"):
        Mx4RequestCachePool([_source(device, 4, 2, 2, 96, "plain", 0)], 8)
    wrong = _source(device, 4, 2, 2, 64, "plain", 0)
    wrong.layers[1].values = wrong.layers[1].values.float()
    with pytest.raises(ValueError, match="bf16"):
        Mx4RequestCachePool([good, wrong], 8)
    wrong.layers[1].values = wrong.layers[1].values[:, :1].to(torch.bfloat16)
    with pytest.raises(ValueError, match="Hkv"):
        Mx4RequestCachePool([good, wrong], 8)


def _setup(device, transformers):
    """A wave of five requests over a 4-bit pool, and over a bf16 pool of the values
    that the 4-bit one holds."""
    from specgrove_amd.cache import Mx4RequestCachePool, PersistentRequestCachePool
    cpu_model, gpu_model, stack = stack_cases._tiny_models(transformers, device)
    rng = np.random.default_rng(12)
    prompts = [rng.integers(0, 4096, size=int(rng.integers(24, 90))) for _ in range(5)]
    few = Mx4RequestCachePool(stack_cases._prefill(cpu_model, prompts, device), capacity=160)
    same = PersistentRequestCachePool(
        [_Cache([_Layer(layer.keys, layer.values) for layer in c.layers]) for c in few.caches],
        capacity=160)
    parents = [W.random_parent_tree(int(n), rng, max_depth=6) for n in (16, 9, 1, 24, 12)]
    blocks = [SimpleNamespace(nodes=list(range(len(p))), parents=p,
                              tokens=W.random_tokens(p, 4096, rng), depths=W.depths_of(p))
              for p in parents]
    return SimpleNamespace(cpu_model=cpu_model, gpu_model=gpu_model, stack=stack, few=few,
                           same=same, prompts=prompts, parents=parents, blocks=blocks)


def _run(s, runner, pool, device):
    from specgrove_amd import attention
    from specgrove_amd.cache import pack_cache_sequence
    lengths = list(pool.lengths)
    offsets = list(np.cumsum([0] + lengths[:-1]))
    states = [SimpleNamespace(generated=[int(s.prompts[i][-1])], block_root=0, tree=None,
                              round_prefix_len=lengths[i], target_cache=pool.caches[i])
              for i in range(5)]
    ids, positions, mask, qoff = attention.pack_block_inputs(
        states, s.blocks, lengths, offsets, sum(lengths), torch.bfloat16, device)
    packed, _, _, total = pack_cache_sequence(pool.caches)
    with torch.no_grad():
        out = runner(input_ids=ids, position_ids=positions, attention_mask=mask,
                     past_key_values=packed, use_cache=True, output_hidden_states=True)
    return out, packed, qoff, total, (ids, positions, lengths)


def _reference(s, inputs, pool):
    """The wave in fp32 on the CPU over the pool's values."""
    from transformers import DynamicCache
    ids, positions, lengths = inputs
    model = copy.deepcopy(s.cpu_model).float()
    model.config._attn_implementation = "sdpa"
    cache = DynamicCache()
    for layer in range(2):
        cache.update(
            torch.cat([pool.caches[i].layers[layer].keys.float().cpu() for i in range(5)], 2),
            torch.cat([pool.caches[i].layers[layer].values.float().cpu() for i in range(5)], 2),
            layer)
    dense = torch.from_numpy(stack_cases.oracle_mask(lengths, s.parents))
    with torch.no_grad():
        return model.model(input_ids=ids.cpu(), position_ids=positions.cpu(),
                           attention_mask=dense[None, None], past_key_values=cache,
                           use_cache=True).last_hidden_state[0]


@pytest.mark.parametrize("through", ["stack", "transformers"])
def test_a_wave_over_the_4_bit_pool(device, through):
    transformers = pytest.importorskip("transformers")
    s = _setup(device, transformers)
    runner = s.stack.model if through == "stack" else s.gpu_model.model
    want = None
    errors = []
    for pool in (s.few, s.same):
        out, packed, qoff, total, inputs = _run(s, runner, pool, device)
        want = _reference(s, inputs, pool) if want is None else want
        errors.append((out.last_hidden_state[0].float().cpu() - want).abs())
        # Commit a path of every request; the pool holds exactly those rows.
        keep = [[0] + ([1] if len(p) > 1 else []) for p in s.parents]
        before = list(pool.lengths)
        pool.append_packed_sequence(packed, pool.caches, total, qoff, keep, device)
        pool.check_status()
        for i, rows in enumerate(keep):
            assert pool.lengths[i] == before[i] + len(rows)
            at = torch.tensor([qoff[i] + r for r in rows], device=device)
            for layer in range(2):
                view, tree = pool.caches[i].layers[layer], packed.layers[layer]
                for got, new in ((view.keys, tree.keys), (view.values, tree.values)):
                    new = new[:, :, at]
                    held = _held(new) if pool is s.few else new.cpu()
                    assert torch.equal(got[:, :, before[i]:].cpu(), held)
    few, same = errors
    print(f"mean {few.mean():.3e} / {same.mean():.3e}, max {few.max():.3e} / {same.max():.3e}",
          flush=True)
    assert few.mean() <= 1.25 * same.mean() + 1e-4
    assert few.max() <= 0.125


def test_commit_refusals_leave_the_pool_as_it_was(device):
    transformers = pytest.importorskip("transformers")
    s = _setup(device, transformers)
    pool = s.few
    _, packed, qoff, total, _ = _run(s, s.stack.model, pool, device)
    before = list(pool.lengths)
    codes = [t.clone() for t in pool._arena]
    with pytest.raises(ValueError, match="disagree"):
        pool.append_packed_sequence(packed, pool.caches, total + 1, qoff, [[0]] * 5, device)
    with pytest.raises(ValueError, match="disagree"):
        pool.append_packed_sequence(packed, pool.caches, total, qoff, [[99]] + [[0]] * 4, device)
    packed.layers[1].values = packed.layers[1].values.float()
    with pytest.raises(ValueError, match="bf16"):
        pool.append_packed_sequence(packed, pool.caches, total, qoff, [[0]] * 5, device)
    pool.capacity = max(before)
    packed.layers[1].values = packed.layers[1].values.to(torch.bfloat16)
    with pytest.raises(RuntimeError, match="capacity exhausted"):
        pool.append_packed_sequence(packed, pool.caches, total, qoff, [[0]] * 5, device)
    assert pool.lengths == before
    assert all(torch.equal(a, b) for a, b in zip(codes, pool._arena))


def test_e4m3_projections_are_the_operators_one_by_one(device):
    """Stack(projections="fp8") over the 4-bit pool: bit for bit the public operators
    in sequence, and near the bf16 stack over the weights that were packed."""
    transformers = pytest.importorskip("transformers")
    from specgrove_amd import attention, ops, target
    s = _setup(device, transformers)
    stack = target.Qwen3TargetStack.from_transformers(s.gpu_model, projections="fp8")
    out, packed, _, _, (ids, positions, _) = _run(s, stack.model, s.few, device)
    mask = attention.build_tree_mask(s.few, s.few.caches, s.parents, device)
    plan = mask.plan(4, 2, 64)
    rows = ids.shape[1]
    x = torch.nn.functional.embedding(ids[0], stack.embed)
    carry, residual = x, None
    for index, layer in enumerate(stack.layers):
        h, residual = target.add_rmsnorm_fp8(carry, layer.ln1, stack.eps, residual,
                                             want_sum=True)
        q, k, v = target.qk_norm_rope(ops.fp8_matmul(h, layer.wqkv), 4, 2, 64, layer.q_norm,
                                      layer.k_norm, stack.inv_freq, positions.reshape(-1),
                                      stack.eps)
        a = ops.tree_attention_mx4(
            q, s.few.k_codes[index], s.few.k_scales[index], s.few.v_codes[index],
            s.few.v_scales[index], k.transpose(0, 1), v.transpose(0, 1), mask.row_offset,
            mask.prefix_start, mask.prefix_len, mask.parent, plan)
        o = ops.fp8_matmul(ops.quantize_fp8(a.view(rows, -1)), layer.wo)
        h, residual = target.add_rmsnorm_fp8(o, layer.ln2, stack.eps, residual, want_sum=True)
        carry = ops.fp8_matmul(target.silu_mul_fp8(ops.fp8_matmul(h, layer.wgu)), layer.wd)
        assert torch.equal(packed.layers[index].keys[0], k)
    final = target.add_rmsnorm(carry, stack.norm, stack.eps, residual)
    assert torch.equal(out.last_hidden_state[0], final)

    # The same weights in bf16: 8 products, each row off by at most 2^-4 of its norm.
    rounded = copy.deepcopy(s.gpu_model)

    def unpacked(*parts):
        codes, scales = ops.quantize_fp8_weight(torch.cat([p.weight for p in parts], 0))
        grid = scales.repeat_interleave(128, 0).repeat_interleave(128, 1)
        values = codes.float() * grid[:codes.shape[0], :codes.shape[1]]
        with torch.no_grad():
            for p, w in zip(parts, values.split([p.weight.shape[0] for p in parts])):
                p.weight.copy_(w)

    for layer in rounded.model.layers:
        a, m = layer.self_attn, layer.mlp
        unpacked(a.q_proj, a.k_proj, a.v_proj)
        unpacked(a.o_proj)
        unpacked(m.gate_proj, m.up_proj)
        unpacked(m.down_proj)
    plain = target.Qwen3TargetStack.from_transformers(rounded)
    want = _run(s, plain.model, s.few, device)[0].last_hidden_state[0].float()
    off = ((final.float() - want).norm(dim=1) / want.norm(dim=1)).max().item()
    print(f"largest relative difference of a row {off:.3e}", flush=True)
    assert off <= 8 * 2.0 ** -4


def test_stack_refuses_unknown_projections(device):
    transformers = pytest.importorskip("transformers")
    from specgrove_amd import target
    _, gpu_model, _ = stack_cases._tiny_models(transformers, device)
    with pytest.raises(ValueError, match="projections"):
        target.Qwen3TargetStack.from_transformers(gpu_model, projections="int8")


peaked = decode_cases.peaked


@pytest.mark.parametrize("model", ["transformers", "stack", "fp8 stack"])
def test_decoding_over_the_4_bit_pool(peaked, device, oracle, model):
    """Whole decodes: every wave's decisions match the oracle sampler on the wave's
    logits, and the lengths add up."""
    from specgrove_amd import target
    from specgrove_amd.cache import Mx4RequestCachePool
    gpu_model, cpu_model, prompts = peaked
    runner = gpu_model
    if model != "transformers":
        runner = target.Qwen3TargetStack.from_transformers(
            gpu_model, projections="fp8" if model == "fp8 stack" else "bf16")
    drafter = decode_cases._Drafter(cpu_model, prompts)
    result, waves, states = decode_cases._decode(
        (runner, cpu_model, prompts), device, oracle, persistent=True, drafter=drafter,
        max_new=16, row_cap=16, cache_format="mx4")
    assert all(isinstance(s.target_cache.pool, Mx4RequestCachePool) for s in states)
    assert len(result.outputs) == len(prompts) and len(waves) == result.physical_target_calls
