"""The cache of device work lists (host logic, no GPU): least recently used entries go, those a captured graph was given
stay, and threads may use it at once."""
import threading

import pytest
import torch


@pytest.fixture(scope='module', autouse=True)
def _library():
    from onereel_b200.csrc.build import build
    build()


def test_evicts_the_least_recently_used_half():
    from onereel_b200.attention import _Plans
    c, made = _Plans(limit=8), []

    def get(k):
        return c.get(k, 'cpu', lambda: made.append(k) or (torch.full((1,), k), 1))
    for k in range(8):
        get(k)
    assert get(0)[0].item() == 0 and made == list(range(8))
    get(8)                                            # one too many: the newest four stay, 0 among them
    assert list(c.entries) == [6, 7, 0, 8]
    get(1)
    assert made == [*range(9), 1]


def test_what_a_captured_graph_was_given_stays(monkeypatch):
    from onereel_b200 import attention as A
    c = A._Plans(limit=4)
    first = c.get('a', 'cpu', lambda: (torch.zeros(1), 1))
    monkeypatch.setattr(A, 'capturing', lambda device: True)
    assert c.get('a', 'cpu', None) is first
    monkeypatch.setattr(A, 'capturing', lambda device: False)
    for k in range(50):
        c.get(k, 'cpu', lambda: (torch.zeros(1), 1))
    assert 'a' not in c.entries and c.held['a'] is first
    assert c.get('a', 'cpu', None) is first           # and is used again, not built twice


def test_work_lists_come_from_the_cache(monkeypatch):
    from onereel_b200 import attention as A
    monkeypatch.setattr(A, '_PLANS', A._Plans(limit=6))
    monkeypatch.setattr(A, '_BWD_PLANS', A._Plans(limit=6))
    fwd = A.plan([0], [5], [0], [7], 2, 'cpu')
    bwd = A._plan_bwd([0], [5], [0], [7], 2, 5, 7, 'cpu')
    assert A.plan([0], [5], [0], [7], 2, 'cpu') is fwd and A._plan_bwd([0], [5], [0], [7], 2, 5, 7, 'cpu') is bwd
    assert fwd[1] == 2 and bwd[2] == 4                # one item per head; a query and a key item per head
    for n in range(1, 20):
        A.plan([0], [n], [0], [7], 2, 'cpu')
        A._plan_bwd([0], [n], [0], [7], 2, n, 7, 'cpu')
    assert len(A._PLANS.entries) <= 6 and len(A._BWD_PLANS.entries) <= 6


def test_threads():
    from onereel_b200.attention import _Plans
    c, errors = _Plans(limit=4), []

    def work(seed):
        try:
            for i in range(3000):
                k = (i * (seed + 3)) % 9
                assert c.get(k, 'cpu', lambda: (torch.full((1,), k), k))[1] == k
        except Exception as e:                        # noqa: BLE001 (reported below)
            errors.append(e)
    ts = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors


def test_tables_are_refused_during_a_capture(monkeypatch):
    """the error comes before the copy that would end the capture, and says what to do"""
    from onereel_b200 import attention as A, pack
    monkeypatch.setattr(pack, 'capturing', lambda device: True)
    monkeypatch.setattr(A, '_PLANS', A._Plans())
    monkeypatch.setattr(A, '_BWD_PLANS', A._Plans())
    for call in (lambda: A.plan([0], [3], [0], [4], 1, 'cpu'), lambda: A._plan_bwd([0], [3], [0], [4], 1, 3, 4, 'cpu'),
                 lambda: pack.RunTable([0], [0], [0], [0], [64], 'cpu'), lambda: pack.RowSum([0], [0], 1, 'cpu')):
        with pytest.raises(RuntimeError, match='once before capturing'):
            call()
    assert not A._PLANS.entries and not A._BWD_PLANS.entries


def test_work_lists_know_the_rows_they_need():
    """the ends of the segments that have queries, and of their keys; empty ones need nothing"""
    from onereel_b200 import attention as A
    for segs, need in ((([0, 9], [5, 3], [4, 0], [6, 30]), (12, 30)), (([7], [2], [50], [0]), (9, 0)),
                       (([0, 90], [5, 0], [0, 70], [8, 9]), (5, 8)), (([], [], [], []), (0, 0))):
        assert A.plan(*segs, 2, 'cpu')[2:] == need
