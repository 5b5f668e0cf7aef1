"""BatchDecoder over a quantized K/V cache (qmk_batch_forward_kvq) against the
torch-fp32 oracle.

The oracle attends to the rows that the decoder's cache holds, and checks each
against its own K or V row: off by at most half a code step, s / 2 with s the
group's largest magnitude / 7 or / 127, s itself rounded to bf16 (2^-8 of it),
and by what the two evaluations differ by before they round (their fp32 rows
agree to 2^-17 of the activations; 5e-3 is allowed).  The oracle cannot round
for itself: a value within that difference of the border of two codes falls on
either side, and in a sequence of 5 tokens one V element off by a code step
(0.3 of a row of order 1) moves x by 0.2 * 0.3 * 0.02 in each of 1024 elements,
0.04 of |x| ~ 1, and so the logits by 0.04 * 32 * 0.02 = 0.026, past the
tolerances that hold for everything else (logits within 2e-2, mean 1.5e-3,
rel-L2 5e-3)."""

import pytest
import torch

from test_gpu_parity import V, _check_vs_oracle, small_model

pytestmark = pytest.mark.gpu


class HeldCache:
    """A cache tensor of MirrorDecoder: the rows [layers, heads, positions,
    head_dim] that the decoder holds, checked against those that are set."""

    dtype = torch.float32

    def __init__(self, rows, bits):
        self.t, self.top = rows, 7 if bits == 4 else 127

    def __setitem__(self, at, rows):
        g = rows.unflatten(-1, (-1, 32))
        half = g.abs().amax(-1, keepdim=True) / self.top * (0.5 + 2.0**-8 * self.top)
        off = (self.t[at].unflatten(-1, (-1, 32)) - g).abs() - half
        assert off.max().item() < 5e-3, f"a held value is {off.max().item()} past half a step off"

    def __getitem__(self, at):
        return self.t[at]


def oracle(w, bd, seq, tokens):
    """Logits of every position of ``tokens``, sequence ``seq`` of ``bd``."""
    from oracle.qwen3_mirror import MirrorDecoder
    from qwen_megakernel_b200 import KVRows

    m = MirrorDecoder(w, len(tokens), device="cuda", kv_dtype=torch.float32)
    rows = KVRows([0], [len(tokens)], [seq])
    held = [bd.kv.read(rows, layer, dtype=torch.float32) for layer in range(bd.fw.num_layers)]
    m.k_cache, m.v_cache = (HeldCache(torch.stack([h[i].transpose(0, 1) for h in held]), bd.kv.bits) for i in (0, 1))
    return m.prefill(tokens, 0)


def _tokens(n, seed):
    return [int(t) for t in torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed))]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("layers", [1, 2])
def test_quantized_batch_matches_oracle(bits, layers):
    """Prompts of 1 to 200 tokens in one pass (both attention kernels), then
    teacher-forced steps, every sequence against the oracle alone."""
    from qwen_megakernel_b200 import BatchDecoder

    w = small_model(layers, seed=31)
    lens, steps = [5, 200, 1, 40], 4
    bd = BatchDecoder(w, len(lens), max_seq_len=256, use_graphs=False, kv_bits=bits)
    assert bd.decode_mode == "token_parallel" and bd.k_cache is None
    prompts = [_tokens(n, 50 + i) for i, n in enumerate(lens)]
    forced = [_tokens(steps, 70 + i) for i in range(len(lens))]
    pl = torch.empty(len(lens), V, device="cuda")
    first = bd.prefill(prompts, logits=pl)
    outs = []
    for t in range(steps):
        lg = torch.empty(len(lens), V, device="cuda")
        bd.step([f[t] for f in forced], logits=lg)
        outs.append(lg)
    torch.cuda.synchronize()
    bd.check_status()
    for s, n in enumerate(lens):
        ref = oracle(w, bd, s, prompts[s] + forced[s])
        _check_vs_oracle(torch.stack([pl[s]] + [o[s] for o in outs]), ref[n - 1:])
        assert first[s] == int(pl[s].argmax())


def test_quantized_prefill_in_chunks():
    """More prompt rows than one pass takes (4096): sequences cut at the chunk
    border go on where they stopped; a second prompt follows the first."""
    from qwen_megakernel_b200 import BatchDecoder

    w = small_model(1, seed=33, max_seq_len=1024)
    lens = [900, 700, 1000, 800, 950]
    bd = BatchDecoder(w, len(lens), max_seq_len=1024, use_graphs=False, kv_bits=4)
    prompts = [_tokens(n, 90 + i) for i, n in enumerate(lens)]
    more = [_tokens(9, 190 + i) for i in range(len(lens))]
    pl, pl2 = torch.empty(len(lens), V, device="cuda"), torch.empty(len(lens), V, device="cuda")
    bd.prefill(prompts, logits=pl)
    bd.prefill(more, logits=pl2)
    for s in (0, 4):
        ref = oracle(w, bd, s, prompts[s] + more[s])
        _check_vs_oracle(torch.stack([pl[s], pl2[s]]), ref[[lens[s] - 1, lens[s] + 8]])


def test_quantized_graph_equals_eager_and_reset():
    from qwen_megakernel_b200 import BatchDecoder

    w = small_model(2, seed=35)
    prompts = [_tokens(n, 110 + n) for n in (3, 70, 20, 1, 9)]
    outs = []
    for graphs in (True, False):
        bd = BatchDecoder(w, 5, max_seq_len=128, use_graphs=graphs, kv_bits=4)
        for _ in range(2):  # a decoder that was reset answers the same
            first = bd.prefill(prompts)
            outs.append((first, bd.generate(first, 16).cpu()))
            bd.check_status()
            bd.reset()
    for first, log in outs[1:]:
        assert first == outs[0][0] and torch.equal(log, outs[0][1])


def test_quantized_batch_reports_and_refuses():
    from qwen_megakernel_b200 import BatchDecoder, BatchError, BatchForward, KVRows, QuantKVCache

    w = small_model(1, seed=37)
    with pytest.raises(ValueError):
        BatchDecoder(w, 2, kv_bits=3)
    with pytest.raises(ValueError):
        BatchDecoder(w, 4, kv_bits=4, decode="megakernel")
    fw = BatchForward(w, 128)
    cache = QuantKVCache(2, 128, 1)
    dev = dict(dtype=torch.int32, device="cuda")
    tok, seq, pos = torch.tensor([5, 6], **dev), torch.tensor([0, 1], **dev), torch.tensor([3, 128], **dev)
    fw.forward_quantized(cache, KVRows.from_tensors(pos, seq=seq), tok, seq, pos)
    with pytest.raises(BatchError, match="out of range"):
        fw.check_status()
    assert cache.k_codes[0, 0, :, 3].any() and not cache.k_codes[1].any()
    for bad in (QuantKVCache(2, 128, 2), QuantKVCache(2, 128, 1, num_kv_heads=4), QuantKVCache(2, 256, 1)):
        with pytest.raises(ValueError):
            fw.forward_quantized(bad, KVRows([0, 0]), tok, seq, pos)
    with pytest.raises(ValueError):
        fw.forward_quantized(cache, KVRows([0, 0, 0], seq_ids=[0, 1, 1]), tok, seq, pos)
