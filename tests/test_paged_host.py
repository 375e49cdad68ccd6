"""Refusals of the paged cache and the token log-probabilities before any launch, and the paged
cache's bookkeeping of pages, on CPU."""

import pytest
import torch

from analysis_spec_b200 import _lib, _ops
from analysis_spec_b200.build import build
from analysis_spec_b200.paged_cache import PagedKVCache, paged_append, paged_attention, rotation_tables
from analysis_spec_b200.token_logprobs import token_logprobs


@pytest.fixture(scope='module')
def lib():
    build()
    return _lib.load()


S18, S8, P = _lib.i64_array([0] * 18), _lib.i64_array([0] * 8), 16  # pointers that are never followed


def test_append_refuses_on_the_host(lib):
    def call(batch=1, rows=1, heads=2, dim=128, dtype=_lib.BF16, page=16, pages=4, width=2, stride=2, cos=None, sin=None,
             rot=0, rot_positions=0, query=None, out=None, hq=0, interleaved=0, key=P, table=P, starts=P):
        _lib.call('speckv_paged_append', key, P, query, out, P, P, S18, table, stride, width, pages, page, starts, None,
                  None, 0, 0, cos, sin, rot_positions, rot, interleaved, batch, hq, heads, rows, dim, dtype, None)
    for match, kw in (('bad sizes', dict(dim=0)), ('bad sizes', dict(batch=-1)), ('unsupported dtype', dict(dtype=7)),
                      ('query without', dict(query=P)), ('come together', dict(cos=P)),
                      ('rotation of', dict(cos=P, sin=P, rot=130, rot_positions=4)),
                      ('rotation of', dict(cos=P, sin=P, rot=3, rot_positions=4)),
                      ('rotation of', dict(cos=P, sin=P, rot=64)), ('interleaved', dict(interleaved=2)),
                      ('page geometry', dict(page=0)), ('page geometry', dict(pages=0)),
                      ('page table rows', dict(batch=2, stride=1)), ('page table rows', dict(table=None)),
                      ('2\\^31 tokens', dict(batch=1 << 16, rows=1 << 16)), ('null pointer', dict(key=None)),
                      ('null pointer', dict(starts=None)),
                      ('2\\^31 positions', dict(width=1 << 30, stride=1 << 30, page=16))):
        with pytest.raises(_lib.SpecKVError, match=match):
            call(**kw)
    call(batch=0)
    call(rows=0)


def test_attention_refuses_on_the_host(lib):
    def call(batch=1, hq=4, hkv=2, dim=128, dtype=_lib.F16, page=16, q=P, lengths=P):
        _lib.call('speckv_paged_attention', q, P, P, S8, P, 2, 2, 4, page, lengths, P, batch, hq, hkv, dim, 1.0, dtype,
                  None, 0, None)
    for match, kw in (('bad sizes', dict(dim=0)), ('not a multiple', dict(hq=3)), ('unsupported dtype', dict(dtype=-1)),
                      ('page geometry', dict(page=-4)), ('above 256', dict(dim=257)), ('null pointer', dict(q=None)),
                      ('null pointer', dict(lengths=None)), ('2\\^20 sequences', dict(batch=(1 << 20) + 1))):
        with pytest.raises(_lib.SpecKVError, match=match):
            call(**kw)
    call(batch=0)


def test_logprobs_refuse_on_the_host(lib):
    def call(batch=1, per=2, source=2, vocab=10, inv_t=1.0, top=0, dtype=_lib.F32, tokens=P, logprobs=P, tops=None,
             rows=None):
        _lib.call('speckv_token_logprobs', P, dtype, 0, 0, tokens, 0, 0, rows, 0, 0, batch, per, source, vocab, inv_t,
                  top, logprobs, P, P, tops, tops, None)
    for match, kw in (('bad sizes', dict(vocab=0)), ('unsupported dtype', dict(dtype=9)), ('temperature', dict(inv_t=0.0)),
                      ('temperature', dict(inv_t=float('nan'))), ('temperature', dict(inv_t=float('inf'))),
                      ('alternatives', dict(top=11)), ('alternatives', dict(top=33, vocab=100)),
                      ('null pointer', dict(top=3)), ('null pointer', dict(tokens=None)),
                      ('null pointer', dict(logprobs=None)), ('rows of logits', dict(source=3)),
                      ('2\\^31 rows', dict(batch=1 << 20, per=1 << 20, source=1 << 20))):
        with pytest.raises(_lib.SpecKVError, match=match):
            call(**kw)
    call(batch=0)

    def back(entropy=P, g_top=None, top=0, ids=None, g_lp=P, tokens=P):
        _lib.call('speckv_token_logprobs_backward', P, _lib.F32, 0, 0, tokens, 0, 0, 1, 2, 10, 1.0, top, entropy, P, ids,
                  g_lp, None, g_top, P, None)
    for kw in (dict(entropy=None), dict(g_top=P), dict(g_top=P, top=2), dict(tokens=None)):
        with pytest.raises(_lib.SpecKVError, match='null pointer'):
            back(**kw)


def test_front_end_refuses_cpu_tensors():
    x = torch.zeros(2, 2, 1, 128)
    pool, table, n = torch.zeros(4, 2, 16, 128), torch.zeros(2, 2, dtype=torch.long), torch.zeros(2, dtype=torch.long)
    for go in (lambda: paged_append(x, x, pool, pool, table, n), lambda: paged_attention(x, pool, pool, table, n),
               lambda: token_logprobs(torch.zeros(2, 5), n)):
        with pytest.raises(RuntimeError, match='no CPU path'):
            go()


def test_score_operands_are_checked():
    """Shapes, dtypes and ranges are refused before the device is looked at."""
    x, t = torch.zeros(3, 7), torch.zeros(3, dtype=torch.long)
    for match, kw in (('dtype', dict(logits=x.double())), ('unit stride', dict(logits=torch.zeros(7, 3).T)),
                      ('vocabulary', dict(logits=torch.zeros(1, 1, 3, 7))), ('vocabulary', dict(logits=x[0, 0])),
                      ('alternatives', dict(top=8)), ('alternatives', dict(top=-1)),
                      ('temperature', dict(temperature=0.0)), ('temperature', dict(temperature=-1.0)),
                      ('temperature', dict(temperature=float('nan'))), ('temperature', dict(temperature=float('inf'))),
                      ('tokens', dict(tokens=t[:2])), ('tokens', dict(tokens=t.int())), ('rows', dict(rows=t[None])),
                      ('rows', dict(logits=x[None], rows=t)), ('tokens', dict(logits=x[None], rows=t[None])),
                      ('carries no gradient', dict(logits=torch.zeros(1, 3, 7, requires_grad=True), rows=t[None],
                                                   tokens=t[None]))):
        with pytest.raises(ValueError, match=match):
            token_logprobs(**{'logits': x, 'tokens': t, **kw})


def test_paged_operands_are_checked():
    bf = torch.bfloat16
    good = dict(key=torch.zeros(2, 2, 3, 64, dtype=bf), value=torch.zeros(2, 2, 3, 64, dtype=bf),
                key_pages=torch.zeros(4, 2, 16, 64, dtype=bf), value_pages=torch.zeros(4, 2, 16, 64, dtype=bf),
                page_table=torch.zeros(2, 2, dtype=torch.long), starts=torch.zeros(2, dtype=torch.long))
    with pytest.raises(RuntimeError, match='no CPU path'):
        paged_append(**good)
    q, n = torch.zeros(2, 4, 3, 64, dtype=bf), torch.zeros(2, dtype=torch.long)
    half = torch.zeros(8, 32)
    for match, kw in (('one shape', dict(value=good['value'][:1])), ('dtype differs', dict(key=good['key'].half())),
                      ('dtype', dict(key=good['key'].double(), value=good['value'].double(),
                                     key_pages=good['key_pages'].double(), value_pages=good['value_pages'].double())),
                      ('one dtype', dict(value_pages=good['value_pages'].half())),
                      ('match the pages', dict(key_pages=good['key_pages'][:, :1], value_pages=good['value_pages'][:, :1])),
                      ('unit stride', dict(key=torch.zeros(2, 2, 64, 3, dtype=bf).transpose(2, 3))),
                      ('unit stride', dict(key_pages=torch.zeros(4, 2, 64, 16, dtype=bf).transpose(2, 3))),
                      ('page table', dict(page_table=n[:, None].int())), ('page table', dict(page_table=n[:1, None])),
                      ('page table', dict(page_table=torch.zeros(2, 2, dtype=torch.long).T)),
                      ('starts', dict(starts=n[:1])), ('starts', dict(starts=n.int())), ('counts', dict(counts=n[:1])),
                      ('positions', dict(positions=n[:, None])), ('positions', dict(positions=torch.zeros(2, 3))),
                      ('rotation', dict(rotation=(half, half[:4]))), ('rotation', dict(rotation=(half.half(), half.half()))),
                      ('rotation', dict(rotation=(half.T, half.T))), ('rotation', dict(rotation=(half, None))),
                      ('rotation of 66', dict(rotation=(torch.zeros(8, 33),) * 2)),
                      ('rotation of 64', dict(rotation=(half[:0], half[:0]))),
                      ('query must', dict(query=q[:, :, :2])), ('query must', dict(query=q.half())),
                      ('one shape and dtype', dict(query=q, query_out=q[:, :2])),
                      ('without query', dict(query_out=q))):
        with pytest.raises(ValueError, match=match):
            paged_append(**{**good, **kw})
    good = dict(query=q[:, :, :1], key_pages=good['key_pages'], value_pages=good['value_pages'],
                page_table=good['page_table'], lengths=n)
    with pytest.raises(RuntimeError, match='no CPU path'):
        paged_attention(**good)
    for match, kw in (('one new token', dict(query=q)), ('match the pages', dict(query=q[:, :3, :1])),
                      ('match the pages', dict(query=q[:, :, :1, :32])), ('match the pages', dict(query=q[:, :, :1].half())),
                      ('lengths', dict(lengths=n[:1])), ('out must', dict(out=q[:, :, :1])),
                      ('out must', dict(out=torch.zeros(2, 1, 4, 64))),
                      ('unit stride', dict(query=torch.zeros(2, 4, 64, 2, dtype=bf).transpose(2, 3)[:, :, :1]))):
        with pytest.raises(ValueError, match=match):
            paged_attention(**{**good, **kw})


def test_page_bookkeeping(monkeypatch):
    """Pages handed out and back, table and lengths on the device, refusals that change nothing."""
    cache = PagedKVCache(8, 4, batch_capacity=3, max_length=20)
    with pytest.raises(ValueError, match='batch capacity'):
        cache.admit(4)
    assert cache.admit(2) == 0
    cache.begin([5, 9], device='cpu')
    assert cache.lengths == [5, 9] and cache.free_pages == 3
    table = cache.page_table()
    assert table.shape == (2, 5) and len({*table[0, :2].tolist(), *table[1, :3].tolist()}) == 5
    first, starts, counts, lengths = cache._step
    assert (first, starts.tolist(), counts.tolist(), lengths.tolist()) == (0, [0, 0], [5, 9], [5, 9])
    before = cache.page_table().clone()
    cache.begin()  # one token each, inside the pages held
    assert cache.lengths == [6, 10] and cache.free_pages == 3 and torch.equal(cache.page_table(), before)
    assert cache._step[1].tolist() == [5, 9]
    assert cache.admit(1) == 2
    with pytest.raises(RuntimeError, match='pages needed'):
        cache.begin([16], first=2)
    with pytest.raises(ValueError, match='max_length'):
        cache.begin([21], first=2)
    with pytest.raises(ValueError, match='token counts'):
        cache.begin([-1], first=2)
    assert cache.lengths == [6, 10, 0] and cache.free_pages == 3
    cache.begin([12], first=2)
    assert cache.free_pages == 0 and cache._step[0] == 2
    last = cache.page_table()[2].tolist()
    assert cache.release([True, False, False]) == [2, 1]
    assert cache.lengths == [12, 10] and cache.free_pages == 2 and cache.page_table()[0].tolist() == last
    with pytest.raises(RuntimeError, match='begin'):
        cache._begun(2)
    with pytest.raises(ValueError, match='entry per live'):
        cache.release([True])
    cache.reset()
    assert cache.free_pages == 8 and cache.statistics()['sequences'] == 0
    assert sorted(cache._free) == list(range(8))
    for bad in ((0, 4, 1, 4), (4, 0, 1, 4), (4, 4, 0, 4), (4, 4, 1, 0)):
        with pytest.raises(ValueError, match='positive'):
            PagedKVCache(bad[0], bad[1], batch_capacity=bad[2], max_length=bad[3])


def test_rotation_tables_hold_far_positions():
    cos, sin = rotation_tables(200001, 64, theta=1e6, device='cpu')
    assert cos.shape == sin.shape == (200001, 32) and cos.dtype == torch.float32
    angle = 200000 * 1e6 ** (-2 * 3 / 64)
    assert abs(cos[200000, 3].item() - __import__('math').cos(angle)) < 1e-6  # fp32 rounding of an exact cosine
    with pytest.raises(ValueError, match='even'):
        rotation_tables(4, 3, device='cpu')


def test_paged_update_refuses_multi_token_steps(monkeypatch):
    """The transformers protocol on CPU, with the launch replaced by a recorder."""
    calls = []
    monkeypatch.setattr(_ops, 'paged_append', lambda *a: calls.append(a))
    cache = PagedKVCache(8, 4, batch_capacity=2, max_length=16)
    k = torch.zeros(2, 1, 3, 8)
    cache.prompt_lengths([3, 1])
    assert cache.update(k, k, 0)[0] is k and cache.update(k, k, 1)[0] is k
    assert cache.lengths == [3, 1] and len(calls) == 2 and calls[0][6].tolist() == [3, 1]
    assert cache.get_seq_length() == 3 and cache.get_mask_sizes(1) == (4, 0) and len(cache) == 2
    with pytest.raises(ValueError, match='one token'):
        cache.update(k, k, 0)
    keys, values = cache.update(k[:, :, :1], k[:, :, :1], 0)
    assert keys.shape == (8, 1, 4, 8) and keys._speckv_pages[1].tolist() == [4, 2]
    assert cache.lengths == [4, 2]
    with pytest.raises(ValueError, match='live request count'):
        cache.update(k[:1, :, :1], k[:1, :, :1], 0)


def test_prompt_lengths_of_one_row(monkeypatch):
    """Prompts whose batch is one row wide have lengths too: an empty one stays empty."""
    calls = []
    monkeypatch.setattr(_ops, 'paged_append', lambda *a: calls.append(a))
    cache = PagedKVCache(8, 4, batch_capacity=2, max_length=16)
    k = torch.zeros(2, 1, 1, 8)
    cache.prompt_lengths([1, 0])
    keys, _ = cache.update(k, k, 0)
    assert cache.lengths == [1, 0] and keys._speckv_pages[1].tolist() == [1, 0] and calls[0][6].tolist() == [1, 0]
    cache.update(k, k, 0)
    assert cache.lengths == [2, 1]
    cache.prompt_lengths([1])
    with pytest.raises(ValueError, match='prompt lengths'):
        cache.update(k, k, 0)


def test_negative_strides_are_refused(lib):
    with pytest.raises(_lib.SpecKVError, match='negative stride'):
        _lib.call('speckv_paged_append', P, P, None, None, P, P, _lib.i64_array([0] * 17 + [-16]), P, 2, 2, 4, 16, P, None,
                  None, 0, 0, None, None, 0, 0, 0, 1, 0, 2, 1, 128, _lib.BF16, None)
    with pytest.raises(_lib.SpecKVError, match='negative stride'):
        _lib.call('speckv_paged_attention', P, P, P, _lib.i64_array([0, 0, -1, 0, 0, 0, 0, 0]), P, 2, 2, 4, 16, P, P, 1, 2, 2,
                  128, 1.0, _lib.BF16, None, 0, None)


def test_prompt_lengths_hold_for_one_forward(monkeypatch):
    """A forward that fails takes its prompt lengths and the sequences it admitted with it, and leaves none begun."""
    monkeypatch.setattr(_ops, 'paged_append', lambda *a: None)
    cache = PagedKVCache(16, 4, batch_capacity=3, max_length=24)
    k = torch.zeros(3, 1, 20, 8)
    cache.prompt_lengths([7, 20])
    with pytest.raises(ValueError, match='prompt lengths'):
        cache.update(k, k, 0)
    assert cache.lengths == [] and cache.free_pages == 16
    cache.update(k, k, 0)
    assert cache.lengths == [20, 20, 20]
    cache.reset()
    cache.prompt_lengths([7, 25, 13])
    with pytest.raises(ValueError, match='max_length'):  # fails in begin
        cache.update(torch.zeros(3, 1, 30, 8), torch.zeros(3, 1, 30, 8), 0)
    assert cache.lengths == [] and cache.free_pages == 16
    cache.update(k[:2], k[:2], 0)  # a smaller batch, every row of it live
    assert cache.lengths == [20, 20]
    cache.prompt_lengths([7, 20, 13])
    cache.reset()
    cache.update(k, k, 0)
    assert cache.lengths == [20, 20, 20]
    with pytest.raises(RuntimeError, match='pages needed'):
        cache.update(k[:, :, :1], k[:, :, :1], 0)
    assert cache.lengths == [20, 20, 20]
    with pytest.raises(RuntimeError, match='begin'):
        cache.append(k[:, :, :1], k[:, :, :1], 0)


def test_append_needs_the_begun_rows(monkeypatch):
    """Fewer rows than begun would leave positions that count as stored and hold nothing."""
    calls = []
    monkeypatch.setattr(_ops, 'paged_append', lambda *a: calls.append(a))
    cache = PagedKVCache(16, 4, batch_capacity=2, max_length=24)
    cache.admit(2)
    cache.begin([2, 5], device='cpu')
    k = torch.zeros(2, 1, 4, 8)
    with pytest.raises(ValueError, match='4 rows for a forward begun over up to 5'):
        cache.append(k, k, 0)
    assert not calls
    wide = torch.zeros(2, 1, 6, 8)  # padding behind the longest is the callers' choice
    cache.append(wide, wide, 0)
    cache.begin(1)
    cache.append(k[:, :, :1], k[:, :, :1], 0)
    assert len(calls) == 2


def test_a_step_lies_in_the_same_memory_each_time(monkeypatch):
    """Table, starts, counts and lengths keep their addresses, which a captured step has recorded; what
    happens on the host is refused inside a capture, and changes nothing."""
    cache = PagedKVCache(16, 4, batch_capacity=4, max_length=40)
    cache.admit(2)
    cache.begin([5, 9], device='cpu')
    cache.begin()
    step = cache._step
    places = [t.data_ptr() for t in (*step[1:], cache.page_table())]
    assert cache.admit(1) == 2
    cache.begin([3], first=2)
    assert cache.release([False, False, True]) == [0, 1]
    for i in range(5):
        cache.begin()
        assert [t.data_ptr() for t in (*cache._step[1:], cache.page_table())] == places
        assert [t.tolist() for t in step[1:]] == [[6 + i, 10 + i], [1, 1], [7 + i, 11 + i]]
    cache._device = torch.device('cuda')  # as if the pools were on a GPU whose stream is being captured
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    before = cache.lengths[:], cache.free_pages
    for refused in (cache.begin, lambda: cache.release([True, False])):
        with pytest.raises(RuntimeError, match='not inside its capture'):
            refused()
    assert (cache.lengths, cache.free_pages) == before


def test_cache_operations_on_rows_are_refused(monkeypatch):
    """transformers' own forms of these pass over a cache without layer objects and change nothing."""
    monkeypatch.setattr(_ops, 'paged_append', lambda *a: None)
    cache = PagedKVCache(8, 4, batch_capacity=2, max_length=16)
    k = torch.zeros(2, 1, 3, 8)
    cache.update(k, k, 0)
    for call in (lambda: cache.crop(2), lambda: cache.reorder_cache(torch.tensor([1, 0])),
                 lambda: cache.batch_repeat_interleave(2), lambda: cache.batch_select_indices(torch.tensor([0]))):
        with pytest.raises(NotImplementedError, match='admit, release'):
            call()
    assert cache.lengths == [3, 3]


def test_profile_events_go_to_the_operands_gpu(monkeypatch):
    """The front end launches on its operands' GPU; events of the current one would time nothing."""
    class Device:
        now = 0

        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, Device.now = Device.now, self.index

        def __exit__(self, *error):
            Device.now = self.before

    class Event:
        def __init__(self, enable_timing):
            self.at = None

        def record(self):
            self.at = Device.now

    class Front:
        def paged_attention(self, *args):
            return Device.now

    monkeypatch.setattr(torch.cuda, 'device', Device)
    monkeypatch.setattr(torch.cuda, 'Event', Event)
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: Device.now)
    monkeypatch.setattr(_lib, 'front', Front)
    monkeypatch.setattr(_ops, '_first_device', lambda values: 1)
    monkeypatch.setattr(_lib.profile, 'enabled', True)
    monkeypatch.setattr(_lib.profile, 'events', {})
    monkeypatch.setattr(_lib.profile, 'calls', 0)
    assert _ops._front('paged_attention', None) == 1 and Device.now == 0
    assert [(s.at, e.at) for s, e in _lib.profile.events['speckv_paged_attention']] == [(1, 1)]


def test_tangents_are_refused():
    from torch.autograd import forward_ad
    x, t = torch.zeros(3, 7), torch.zeros(3, dtype=torch.long)
    with forward_ad.dual_level():
        for logits in (forward_ad.make_dual(x, x + 1), forward_ad.make_dual(x.requires_grad_(True), x + 1)):
            with pytest.raises(ValueError, match='forward-mode'):
                token_logprobs(logits, t)
    with pytest.raises(RuntimeError, match='no CPU path'):
        token_logprobs(x, t)


def test_a_first_forward_inside_a_capture_leaves_nothing(monkeypatch):
    """Refused with its reason, and the sequences it admitted are gone."""
    monkeypatch.setattr(_ops, 'paged_append', lambda *a: None)
    cache = PagedKVCache(8, 4, batch_capacity=2, max_length=16)
    k = torch.zeros(2, 1, 3, 8)
    cache.update(k, k, 0)
    cache.reset()
    assert cache.free_pages == 8 and cache.lengths == []
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
        m.setattr(cache, '_device', torch.device('cuda'))
        with pytest.raises(RuntimeError, match='begin.. decides and copies'):
            cache.update(k, k, 0)
    assert cache.free_pages == 8 and cache.lengths == []
    cache.update(k, k, 0)
    assert cache.lengths == [3, 3] and cache.free_pages == 6


def test_append_refuses_to_write_expanded_tensors():
    bf = torch.bfloat16
    k, n = torch.zeros(2, 2, 3, 64, dtype=bf), torch.zeros(2, dtype=torch.long)
    good = dict(key=k, value=k, key_pages=torch.zeros(4, 2, 16, 64, dtype=bf), value_pages=torch.zeros(4, 2, 16, 64, dtype=bf),
                page_table=torch.zeros(2, 2, dtype=torch.long), starts=n, query=k)
    one = good['key_pages'][:1].expand(4, 2, 16, 64)
    for kw in (dict(key_pages=one), dict(value_pages=one), dict(query_out=k[:1].expand(2, 2, 3, 64))):
        with pytest.raises(ValueError, match='overlap themselves'):
            paged_append(**{**good, **kw})
    for kw in (dict(key=k[:1].expand(2, 2, 3, 64)), dict(query=k[:, :1].expand(2, 4, 3, 64)), dict(query_out=k)):
        with pytest.raises(RuntimeError, match='no CPU path'):  # read only, or in place
            paged_append(**{**good, **kw})


@pytest.mark.parametrize('first', [True, False])
def test_begin_inside_and_outside_inference_mode(first):
    """What one mode has made, a begin in the other writes to."""
    cache = PagedKVCache(16, 4, batch_capacity=2, max_length=24)
    cache.admit(2)
    for mode in (first, not first, first):
        with torch.inference_mode(mode):
            cache.begin([3, 5], device='cpu')
    assert cache._step[3].tolist() == [9, 15] and cache.page_table()[:, 0].tolist() != [0, 0]
    with torch.inference_mode(first):
        assert cache.release([True, False]) == [1]
    cache.begin(4)
    assert cache._step[3].tolist() == [19]


def test_masks_in_inference_mode(monkeypatch):
    """Masks made in inference mode have no version: a prompt's mask keeps its bits all the same, another one is
    converted again for each layer rather than trusted to be unchanged."""
    from analysis_spec_b200 import tree_attention
    made = []

    monkeypatch.setattr(_ops, 'mask_bits', lambda mask, bits, first, flag: (made.append(mask), flag.zero_()))
    with torch.inference_mode():
        query = torch.zeros(2, 4, 5, 128, dtype=torch.bfloat16)
        prompt = {}
        masks = [tree_attention.prompt_mask(prompt, query) for _ in range(3)]
        assert masks[0] is masks[1] and masks[0][1, 0].isfinite().all() and masks[0][0, 0, 1, 2] < -1e38
        for mask in masks:
            assert tree_attention.dense_mask_visibility(mask, mask, 2, 5, 5) is not None
        assert len(made) == 1
        other = torch.zeros(2, 1, 5, 5, dtype=torch.bfloat16)
        for _ in range(2):
            assert tree_attention.dense_mask_visibility(other, other, 2, 5, 5) is not None
        assert len(made) == 3
