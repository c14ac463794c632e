"""The cache's operators captured into CUDA graphs: a decoding step that is replayed token by token, an eviction, the prompts; alone, on another
stream, and next to another graph of the same operators."""
import pytest
import torch

pytestmark = pytest.mark.gpu

KINDS = [(torch.bfloat16, 8, 2, 128, 16), (torch.float16, 4, 4, 64, 64), (torch.float32, 4, 2, 64, 8), (torch.bfloat16, 6, 3, 33, 7)]
IDS = [f"{str(k[0])[6:]}_{k[1]}x{k[2]}_d{k[3]}_p{k[4]}" for k in KINDS]
BLOCK, STEPS, BUDGET = 64, 12, 96


class Loop:
    """Everything a serving process holds: fixed tensors, whose contents every call updates."""

    def __init__(self, kind, seed, lens=(300, 77, 150, 1)):
        dtype, hq, hk, d, page = kind
        g = torch.Generator().manual_seed(seed)
        self.lens0, batch = list(lens), len(lens)

        def normal(*shape):
            return torch.randn(*shape, generator=g).to(dtype).cuda()
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        self.q, self.k, self.v = normal(cu[-1], hq, d), normal(cu[-1], hk, d), normal(cu[-1], hk, d)
        self.cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        blocks = sum(-(-n // BLOCK) for n in lens)
        self.mask = ((torch.rand(hk, blocks, blocks, generator=g) < 0.5) | torch.eye(blocks, dtype=torch.bool)).cuda()
        pages = -(-(max(lens) + STEPS) // page)
        self.table = torch.randperm(batch * pages, generator=g).to(torch.int32).reshape(batch, pages).cuda()
        self.kc, self.vc = (torch.zeros(batch * pages, page, hk, d, dtype=dtype, device="cuda") for _ in "kv")
        self.w = torch.zeros(batch, hk, pages * page, device="cuda")
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.one = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
        self.tokens = [(normal(batch, hq, d), normal(batch, hk, d), normal(batch, hk, d)) for _ in range(STEPS)]
        self.q1, self.k1, self.v1 = (t.clone() for t in self.tokens[0])

    def prompts(self):
        import hbsattn_b200 as hb
        out, lse = self.prompt_out                        # of the prompts' attention, which is not what is captured here
        weights = hb.attention_key_weights(self.q, self.k, lse, self.cu, self.cu, self.mask, BLOCK, BLOCK, True)
        self.w.zero_()
        for b, n in enumerate(self.lens0):
            self.w[b, :, :n] = weights[int(self.cu_list[b]):int(self.cu_list[b + 1])].t()
        self.lens.copy_(hb.append_to_cache(self.k, self.v, self.cu, self.kc, self.vc, self.table, torch.zeros_like(self.lens)))
        return weights

    def step(self):
        import hbsattn_b200 as hb
        self.lens.copy_(hb.append_to_cache(self.k1, self.v1, self.one, self.kc, self.vc, self.table, self.lens))
        return hb.paged_attention(self.q1, self.kc, self.vc, self.table, self.lens, key_weights=self.w)

    def evict(self):
        import hbsattn_b200 as hb
        kept, kept_lens = hb.select_keys(self.w, self.lens, BUDGET, 4, 16)
        hb.compact_cache(self.kc, self.vc, self.table, self.lens, kept, kept_lens, key_weights=self.w)
        self.lens.copy_(kept_lens)
        return kept

    def prepare(self):
        import hbsattn_b200 as hb
        self.cu_list = self.cu.tolist()
        self.prompt_out = hb.HBSAttention_with_lse(self.q, self.k, self.v, self.cu, self.cu, self.mask, BLOCK, BLOCK, True)

    def token(self, i):
        for to, x in zip((self.q1, self.k1, self.v1), self.tokens[i]):
            to.copy_(x)

    def state(self):
        return [self.kc, self.vc, self.w, self.lens]


def run(loop, prompts, step, evict):
    """The whole loop by way of three calls; what every call has returned, and the cache at the end."""
    seen = [prompts().clone()]
    for i in range(STEPS):
        loop.token(i)
        seen.append(step().clone())
        if i == STEPS // 2:
            seen.append(evict().clone())
    return seen + [t.clone() for t in loop.state()]


def capture(loop, stream):
    """Three graphs of the loop's calls, captured without running anything of them."""
    made = []
    for call in (loop.prompts, loop.step, loop.evict):
        graph = torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            out = call()
        made.append((graph, out))

    def replay(graph, out):
        def call():
            graph.replay()
            return out
        return call
    return [replay(*m) for m in made]


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_captured_loop_is_the_eager_one(kind):
    loop = Loop(kind, 1)
    loop.prepare()
    want = run(loop, loop.prompts, loop.step, loop.evict)
    calls = capture(loop, torch.cuda.Stream())
    for _ in range(3):                                    # again and again from the prompts on
        assert same(run(loop, *calls), want)
    assert same(run(loop, loop.prompts, loop.step, loop.evict), want)      # eager calls between replays
    assert same(run(loop, *calls), want)


@pytest.mark.parametrize("kind", KINDS[:3], ids=IDS[:3])
def test_two_captured_loops_side_by_side(kind):
    """On streams of their own, at the same time: graphs share no workspace."""
    loops = [Loop(kind, 2), Loop(kind, 3, lens=(40, 500, 3))]
    want, calls, streams = [], [], [torch.cuda.Stream() for _ in loops]
    for loop, stream in zip(loops, streams):
        loop.prepare()
        want.append(run(loop, loop.prompts, loop.step, loop.evict))
        calls.append(capture(loop, stream))
    torch.cuda.synchronize()
    for _ in range(5):
        seen = [[], []]
        for i in range(-1, STEPS):
            for j, (loop, stream) in enumerate(zip(loops, streams)):
                with torch.cuda.stream(stream):
                    if i < 0:
                        seen[j].append(calls[j][0]().clone())
                        continue
                    loop.token(i)
                    seen[j].append(calls[j][1]().clone())
                    if i == STEPS // 2:
                        seen[j].append(calls[j][2]().clone())
        torch.cuda.synchronize()
        for j, loop in enumerate(loops):
            assert same(seen[j] + loop.state(), want[j])
