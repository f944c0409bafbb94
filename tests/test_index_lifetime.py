"""A KeyIndex does not outlive its pool (no GPU: the library's calls are recorded). On the device the index
names its pool's memory."""
import gc

import pytest

import velokv
from velokv import runtime


class FakeLibrary:
    def __init__(self):
        self.next, self.live, self.log = 1, {}, []

    def create(self, kind, out):
        out._obj.value = self.next
        self.live[self.next] = kind
        self.next += 1
        return 0

    def destroy(self, kind, handle):
        assert self.live.pop(handle.value) == kind
        self.log.append(kind)
        return 0

    def vk_pool_create(self, ctx, desc, out):
        return self.create("pool", out)

    def vk_pool_get_desc(self, pool, out):
        return 0

    def vk_index_create(self, ctx, pool, out):
        assert self.live[pool.value] == "pool"
        return self.create("index", out)

    def vk_pool_destroy(self, h):
        return self.destroy("pool", h)

    def vk_index_destroy(self, h):
        return self.destroy("index", h)


class FakeContext:
    h = None


@pytest.fixture
def fake(monkeypatch):
    f = FakeLibrary()
    monkeypatch.setattr(runtime, "lib", lambda: f)
    yield f
    gc.collect()


def pool_of(ctx):
    return velokv.Pool(ctx, 1, 4, 16, 1, 64, velokv.KV_F16)


def test_pool_closed_before_its_indexes(fake):
    ctx = FakeContext()
    pool, other = pool_of(ctx), pool_of(ctx)
    a, b, c = velokv.KeyIndex(ctx, pool), velokv.KeyIndex(ctx, pool), velokv.KeyIndex(ctx, other)
    pool.close()
    assert fake.log == ["index", "index", "pool"]
    assert not a.h and not b.h and c.h  # calls on them are refused: the handle is null
    a.close()
    b.close()
    c.close()
    other.close()
    assert fake.log == ["index", "index", "pool", "index", "pool"] and not fake.live


def test_indexes_go_first_by_themselves(fake):
    ctx = FakeContext()
    pool = pool_of(ctx)
    a = velokv.KeyIndex(ctx, pool)
    a.close()
    b = velokv.KeyIndex(ctx, pool)
    del pool  # the index holds it
    gc.collect()
    assert fake.log == ["index"]
    del a, b
    gc.collect()
    assert fake.log == ["index", "index", "pool"] and not fake.live
