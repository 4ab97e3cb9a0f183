"""Writing many tokens into a 4-bit cache in one call: slots that are named again and again, masked ones, captured calls."""
import numpy as np
import pytest

import fusedmm_amd as fa

pytestmark = pytest.mark.gpu


def operands(t, kv, d, dv, bits, seed):
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n = max(2, t // 3)
    it = torch.int32 if bits == 32 else torch.int64
    slots = torch.randint(-1, n + 1, (t,), generator=gen, device="cuda")      # -1 and n are no slots
    slots[t // 2], slots[-1], slots[0] = n - 1, n - 1, n - 1                  # one slot in the first, a middle and the last place
    ld = kv * d + 8
    k = torch.randn((t, ld), generator=gen, device="cuda").half()
    v = torch.randn((t, kv * dv), generator=gen, device="cuda").half()
    desc = fa.AttnDesc(type=fa.TYPE_F16, maps=1, m=0, n=n, heads=kv, kv_heads=kv, d=d, dv=dv, scale=1.0, ldk=ld, hdk=d, ldv=kv * dv, hdv=dv)
    rec = fa.fusedMM_kv4_record_bytes(1, d, dv)
    return n, slots.to(it), k, v, desc, rec


@pytest.mark.parametrize("t,bits", [(8192, 32), (8193, 64), (30000, 32), (100003, 64)])
def test_the_last_token_of_a_slot_counts_however_many_there_are(t, bits):
    """Against a call that gets each slot's last token alone."""
    import torch
    kv, d, dv = 2, 32, 64
    n, slots, k, v, desc, rec = operands(t, kv, d, dv, bits, seed=t)
    cache, want = [torch.full((n, kv, rec), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(2)]
    assert fa.fusedMM_kv4_write(desc, t, slots, k, v, cache, kv * rec, rec, index_bits=bits) == 0
    host = slots.cpu().numpy()
    last = {int(s): i for i, s in enumerate(host) if 0 <= s < n}
    assert len(last) < t // 2
    order = np.array(sorted(last.items()))
    for a in range(0, len(order), 5000):
        part = order[a:a + 5000]
        at = torch.as_tensor(part[:, 1]).cuda()
        s = torch.as_tensor(part[:, 0]).to(slots.dtype).cuda()
        assert fa.fusedMM_kv4_write(desc, len(part), s, k[at].contiguous(), v[at].contiguous(), want, kv * rec, rec, index_bits=bits) == 0
    torch.cuda.synchronize()
    assert torch.equal(cache, want)


def test_many_tokens_are_captured_and_replayed():
    import torch
    t, kv, d, dv = 20000, 2, 32, 64
    n, slots, k, v, desc, rec = operands(t, kv, d, dv, 32, seed=1)
    cache, want = [torch.zeros((n, kv, rec), dtype=torch.uint8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        assert fa.fusedMM_kv4_write(desc, t, slots, k, v, cache, kv * rec, rec, stream=s.cuda_stream) == 0
    for _ in range(3):
        k.copy_(torch.randn(k.shape, device="cuda"))
        slots.copy_(slots[torch.randperm(t, device="cuda")])
        cache.zero_()
        want.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert fa.fusedMM_kv4_write(desc, t, slots, k, v, want, kv * rec, rec) == 0
        torch.cuda.synchronize()
        assert torch.equal(cache, want)
