"""A beam search as a program runs it: a prompt held once, the beams' own tokens
behind it, and step by step their attention, the choice over beams and vocabulary, the
caches and the next tokens' rows following the choice on the device; against the plain
models doing the same."""
import numpy as np
import pytest

from tests import beam_model
from tests.kv_model import Model, u32s
from tests.test_gpu_kv_attention import compare
from tests.test_gpu_kv_cache import DTYPES, check_read, rows_of
from tests.test_gpu_kv_sequences import KEEP, copied, reordered

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, VOCAB, END = 4, 2, 32, 601, 7


class Decoder:
    """One layer with random weights: rows of a token by table lookup, logits from the
    attention's output."""

    def __init__(self, sdk, dtype, rng):
        self.sdk, self.dtype = sdk, dtype
        t = DTYPES[dtype]
        self.tables = {n: rng.standard_normal((VOCAB, h * DIM)).astype(t) for n, h in (("k", KV), ("v", KV), ("q", HEADS))}
        self.head = (rng.standard_normal((VOCAB, HEADS * DIM)) * 0.4).astype(t)
        self.on_device = {n: sdk.from_numpy(x) for n, x in self.tables.items()}
        self.head_on_device = sdk.from_numpy(self.head)

    def rows(self, tokens, name, count):
        """Rows [batch, heads, 1, DIM] of the tokens' U32 tensor."""
        heads = self.tables[name].shape[1] // DIM
        out = self.sdk.tensor(self.dtype, (count, heads * DIM))
        flat = self.sdk.tensor("u32", (count,))
        self.sdk.lib.tensor_buffer_copy_device(flat.handle, 0, tokens.handle, 0, 4 * count, None, 0)
        self.sdk.call(f"tensor_embedding_lookup_{self.dtype}", self.on_device[name], flat, out)
        shaped = self.sdk.tensor(self.dtype, (count, heads, 1, DIM))
        self.sdk.lib.tensor_buffer_copy_device(shaped.handle, 0, out.handle, 0, out.nbytes, None, 0)
        return shaped


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("groups,beams", [(1, 4), (3, 3)])
def test_beam_search(sdk, groups, beams, dtype):
    rng = np.random.default_rng(groups * beams)
    t, batch, steps = DTYPES[dtype], groups * beams, 8
    decoder = Decoder(sdk, dtype, rng)
    # the prompts, once each
    lengths = [100 + 30 * g for g in range(groups)]
    prompt, prompt_model = sdk.kv_cache(groups, KV, 200, DIM), Model(groups, KV, DIM, DIM)
    k, v = (rows_of(rng, (groups, KV, max(lengths), DIM), dtype) for _ in range(2))
    sdk.call(f"tensor_kv_cache_append_{dtype}", prompt, sdk.from_numpy(k), sdk.from_numpy(v), u32s(lengths))
    prompt_model.append(k, v, lengths)
    own, own_model = sdk.kv_cache(batch, KV, 64 + steps, DIM), Model(batch, KV, DIM, DIM)
    # every beam begins with the same tokens; the first one alone has a score
    before = 61
    k, v = (np.repeat(rows_of(rng, (groups, KV, before, DIM), dtype), beams, 0) for _ in range(2))
    sdk.call(f"tensor_kv_cache_append_{dtype}", own, sdk.from_numpy(k), sdk.from_numpy(v), None)
    own_model.append(k, v)
    first = np.full((groups, beams), -np.inf, np.float32)
    first[:, 0] = 0
    scores, ended = sdk.from_numpy(first), sdk.from_numpy(np.zeros((groups, beams), np.uint32))
    tokens, parents = (sdk.from_numpy(np.full((groups, beams), 3, np.uint32)) for _ in range(2))
    logits = sdk.tensor(dtype, (groups, beams, VOCAB))
    for step in range(steps):
        now = tokens.download().reshape(-1)
        key, value, query = (decoder.rows(tokens, n, batch) for n in ("k", "v", "q"))
        sdk.call(f"tensor_kv_cache_append_{dtype}", own, key, value, None)
        own_model.append(*(decoder.tables[n][now].reshape(batch, KV, 1, DIM) for n in ("k", "v")))
        out = sdk.from_numpy(np.full((batch, HEADS, 1, DIM), 99, t))
        sdk.call(f"tensor_kv_cache_attention_shared_{dtype}", prompt, own, query, None, None, DIM ** -0.5, 1, out)
        compare(beam_model.joined(prompt_model, own_model, [beams] * groups),
                decoder.tables["q"][now].reshape(batch, HEADS, 1, DIM), DIM ** -0.5, True, None, out.download(),
                what=f"step {step}")
        flat, flat_logits = sdk.tensor(dtype, (batch, HEADS * DIM)), sdk.tensor(dtype, (batch, VOCAB))
        sdk.lib.tensor_buffer_copy_device(flat.handle, 0, out.handle, 0, out.nbytes, None, 0)
        sdk.call(f"tensor_linear_{dtype}", flat, decoder.head_on_device, None, flat_logits)
        sdk.lib.tensor_buffer_copy_device(logits.handle, 0, flat_logits.handle, 0, logits.nbytes, None, 0)
        was = [x.download() for x in (logits, scores, ended)]
        sdk.call(f"tensor_beam_select_{dtype}", logits, scores, ended, END, parents, tokens, scores, ended)
        sdk.call("tensor_kv_cache_reorder", own, parents)
        from tests.test_gpu_beam_select import check
        chosen = [x.download() for x in (parents, tokens, scores, ended)]
        check(chosen, *was, END, beams, f"step {step}")
        own_model = reordered(own_model, chosen[0])
        check_read(sdk, own, own_model, f"step {step}")
    # the best beams go on by themselves, their prompts before their own tokens
    best = sdk.kv_cache(groups, KV, 300, DIM)
    sdk.call("tensor_kv_cache_copy", prompt, u32s(range(groups)), best)
    best_model = copied(prompt_model, list(range(groups)), Model(groups, KV, DIM, DIM))
    check_read(sdk, best, best_model, "prompts")
    sdk.call("tensor_kv_cache_copy", own, u32s([g * beams if g else KEEP for g in range(groups)]), best)
    best_model = copied(own_model, [g * beams if g else KEEP for g in range(groups)], best_model)
    check_read(sdk, best, best_model, "own tokens")
