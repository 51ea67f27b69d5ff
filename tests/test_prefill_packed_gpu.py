"""GPU: prefill of prompts of different lengths without padding (orc_prefill_packed, generate_stream(packed=True)) against the left-padded
prefill: logits and the decode that follows within the bf16 tolerance of the stage tests, greedy answers of the chain model equal."""
import pytest
import torch

from conftest import rows_ok
from test_stream_gpu import _batches, chain  # noqa: F401

pytestmark = pytest.mark.gpu


def _prompts(lens, seed, d):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return [(torch.randn(n, d, generator=g, device='cuda') * 0.05).to(torch.bfloat16) for n in lens]


@pytest.mark.parametrize('lens', [[1], [5, 1, 33], [128, 1, 127, 129], [300, 40, 641, 2, 64, 7, 640, 100]], ids=str)
def test_logits_and_decode_agree_with_the_padded_prefill(chain, lens):  # noqa: F811
    from oracle_amd.dims import TINY
    _, eng, _ = chain
    n, d = len(lens), TINY.d_model
    prompts = _prompts(lens, sum(lens), d)
    t = max(lens)
    padded, pos = torch.zeros(n, t, d, dtype=torch.bfloat16, device='cuda'), torch.zeros(n, t, dtype=torch.int32)
    for i, p in enumerate(prompts):
        padded[i, t - lens[i]:] = p
        pos[i, t - lens[i]:] = torch.arange(lens[i], dtype=torch.int32)
    slots, limits = list(range(n))[::-1], [6] * n
    got = []
    for packed in (False, True):
        eng.stream_begin(n)
        if packed:
            first = eng.prefill_packed(slots, torch.cat(prompts), lens, limits, want_logits=True)
        else:
            first = eng.prefill_slots(slots, padded, pos, [t - x for x in lens], limits, want_logits=True)
        for row, slot in enumerate(slots):
            eng.stream_attach(row, slot)
        steps = [eng.decode_step(want_logits=True) for _ in range(2)]
        got.append((first, steps, eng.read_slots()[0]))
    rows_ok(got[1][0], got[0][0], 'packed prefill logits')
    same = (got[0][2][slots, :2] == got[1][2][slots, :2]).all(-1).tolist()       # rows that went on with the same token
    for a, b in zip(got[1][1], got[0][1]):
        keep = [i for i in range(n) if same[i]]
        if keep:
            rows_ok(a[keep], b[keep], 'decode after packed prefill')
    assert sum(same) >= (n + 1) // 2      # random prompts: a near tie may fall either way, not most of them


@pytest.mark.parametrize('n_rows,chunk', [(4, 4), (2, 3)])
def test_packed_stream_gives_the_answers_of_generate(chain, n_rows, chunk):  # noqa: F811
    _, eng, model = chain
    items = _batches([3, 8, 1, 5], seed=20 + n_rows)
    outs = [o.cpu() for o in model.generate_stream(iter(items), max_new_tokens=40, n_rows=n_rows, chunk=chunk, packed=True)]
    assert len(outs) == len(items)
    for k, (item, out) in enumerate(zip(items, outs)):
        ref = model.generate(item['input_ids'], images=item['images'], do_sample=False, use_cache=True, max_new_tokens=40).cpu()
        assert torch.equal(out, ref), k


def test_packed_prefill_refusals(chain):  # noqa: F811
    from oracle_amd import _lib
    from oracle_amd.dims import TINY
    _, eng, _ = chain
    emb = torch.zeros(30, TINY.d_model, dtype=torch.bfloat16, device='cuda')
    eng.prefill(emb[None, :8].contiguous(), torch.arange(8, dtype=torch.int32, device='cuda')[None], [0])
    with pytest.raises(_lib.OracleHipError, match='orc_stream_begin'):
        eng.prefill_packed([0], emb, [30], [4])
    eng.stream_begin(2)
    for slots, lens, limits, text in (([8], [30], [4], 'slot outside'), ([1, 1], [10, 20], [4, 4], 'twice'), ([0, 1], [0, 30], [4, 4], 'prompt length'),
                                      ([0], [30], [49], 'length stop'), ([0], [30], [0], 'length stop')):
        with pytest.raises(_lib.OracleHipError, match=text):
            eng.prefill_packed(slots, emb, lens, limits)
    long = torch.zeros(690, TINY.d_model, dtype=torch.bfloat16, device='cuda')
    with pytest.raises(_lib.OracleHipError, match='max_seq'):
        eng.prefill_packed([0], long, [690], [11])
    eng.prefill_packed([0], long, [690], [10])
    eng.stream_attach(0, 0)
    with pytest.raises(_lib.OracleHipError, match='attached'):
        eng.prefill_packed([0], emb, [30], [4])
    for bad in (lambda: eng.prefill_packed([1], emb, [29], [4]), lambda: eng.prefill_packed([1, 2], emb, [30], [4, 4]), lambda: eng.prefill_packed([1], emb, [30], []),
                lambda: eng.prefill_packed([1], emb[:, :256], [30], [4]), lambda: eng.prefill_packed([1], emb.float(), [30], [4])):
        with pytest.raises(ValueError):
            bad()
