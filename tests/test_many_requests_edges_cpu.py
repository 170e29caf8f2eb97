"""Where a server of many requests meets the rest of the framework: pools that change their size, weights given as variables, threads, layouts that nobody has in mind."""
import pytest
import torch

from dew_b200.inference.serving import Server
from dew_b200.models import CausalTransformer
from dew_b200.nn.kv_cache import KVCache, KVStore

CONFIG = dict(vocab_size=64, emb_features=32, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=16, mlp_features=48, max_seq_len=160)


def model(seed=0, **kw):
    torch.manual_seed(seed)
    return CausalTransformer(**{**CONFIG, **kw}).eval()


# ---------------------------------------------------------------------------------------------------------- pools of another size
def test_a_smaller_pool_leaves_no_name_of_a_page_that_is_gone():
    m = model()
    prompts = [[i % 60 for i in range(49)], [i % 50 for i in range(18)]]
    want = [Server(m, slots=1, capacity=160, kv_cache=KVCache(page_size=8), prefix_cache=False)([p], 6)[0] for p in prompts]
    server = Server(m, slots=2, capacity=160, kv_cache=KVCache(page_size=8), chunk=16)
    server([[1 + i % 50 for i in range(140)], [2 + i % 50 for i in range(130)]], 8)       # names of pages all over the pool
    server.resize(20)
    assert int(server.store.page_table.max()) < 20
    assert server(prompts, 6) == want                         # unequal prompts in several chunks
    server.resize(9)
    short = server.submit(prompts[1], 6)                      # a decode step beside an idle row
    server.run()
    assert short.result() == want[1] and int(server.store.page_table.max()) < 9


def test_a_row_that_lives_through_a_smaller_pool_keeps_its_own_names():
    m, prompt = model(), list(range(3, 30))
    want = Server(m, slots=1, capacity=160, kv_cache=KVCache(page_size=8), prefix_cache=False)([prompt], 20)[0]
    server = Server(m, slots=3, capacity=160, kv_cache=KVCache(page_size=8), chunk=16)
    server([[1 + i % 50 for i in range(140)]] * 3, 8)
    row = server.submit(prompt, 20)
    for _ in range(6):
        server.step()
    before = server.store.page_table.data_ptr()
    server.resize(12)
    assert int(server.store.page_table.max()) < 12 and server.store.page_table.data_ptr() == before
    server.run()
    assert row.result() == want
    server.resize(40)
    assert server([prompt], 20) == [want]


def test_a_store_takes_names_past_its_end_out_of_the_table():
    store = KVStore(KVCache(page_size=8, pages=20), 1, 2, 64, 1, 16, dtype=torch.float32)
    store.page_table.copy_(torch.arange(16, dtype=torch.int32).view(2, 8) + 4)
    store.resize(10)
    assert store.page_table.tolist() == [[4, 5, 6, 7, 8, 9, 0, 0], [0] * 8]
    store.gather(0, 64)
