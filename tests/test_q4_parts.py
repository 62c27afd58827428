"""Which parts a cache of 4 bits takes: what cannot be asked is refused (no GPU)."""
from types import SimpleNamespace

import torch

from nncpu_b200.cache import KVRequest, StateRequest
from nncpu_b200.parts.base import Block, Mixer


class Plain(Mixer):
    def __init__(self, kv=None, state=None, q4=None, shared=False):
        self.kv, self.state, self.shared_kv = kv, state, shared
        if q4 is not None:
            self.takes_q4 = lambda: q4

    def kv_request(self):
        return self.kv

    def state_request(self):
        return self.state


class Of(Block):
    def __init__(self, **parts):
        self.__dict__.update(parts)

    def cache_requests(self):
        return [(KVRequest(2, 64), None)]


KV, STATE = KVRequest(2, 64), StateRequest((8,), torch.float32)


def test_mixers_in_attributes_and_lists():
    a, b = Plain(KV, q4=True), Plain(state=STATE)
    assert Of(mixer=a).takes_q4() and Of(branches=[a, b], again=a).takes_q4()
    assert not Of(mixer=Plain(KV)).takes_q4() and not Of(branches=(a, Plain(KV))).takes_q4()


def test_mixers_that_are_not_found_are_not_taken():
    """A block that asks for keys and values, whose mixers lie where nobody looks."""
    assert not Of(branches={"left": Plain(KV, q4=True)}).takes_q4()
    assert not Of(inner=SimpleNamespace(mixer=Plain(KV))).takes_q4()
    assert Block().takes_q4()               # (asks for nothing)


def test_a_mixer_that_reads_anothers_keys_says_itself_whether_it_can():
    assert Plain(state=STATE).takes_q4() and not Plain(shared=True).takes_q4() and Plain(shared=True, q4=True).takes_q4()
