"""Ranks of the multi-process tests of the operators (gloo, CPU)."""
import os
import traceback


def run_routed_layer(rank, world, port, result_dir):
    """A routed layer with its own router over ``world`` ranks against one rank that holds all experts."""
    import torch
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    torch.set_num_threads(1)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from b200moe.models.layers import MoELayerMulti
        routing = dict(score="sigmoid", groups=4, top_groups=2, group_score=2, balance_bias=True, scale=2.5)
        per_rank = 4
        torch.manual_seed(5)
        whole = MoELayerMulti(32, 48, k=3, num_expert_per_node=per_rank * world, dtype=torch.float32, routing=routing)
        for p in whole.parameters():
            p.data.normal_(0, 0.2)
        whole.expert_bias.normal_(0, 0.1)
        part = MoELayerMulti(32, 48, k=3, num_expert_per_node=per_rank, dtype=torch.float32, dp_group=dist.group.WORLD,
                             routing=routing)
        mine = slice(rank * per_rank, (rank + 1) * per_rank)
        part.router.weight.data.copy_(whole.router.weight)
        part.expert_bias.copy_(whole.expert_bias)
        for name in ("w1", "w2", "w3"):
            getattr(part.experts, name).data.copy_(getattr(whole.experts, name)[mine])
        torch.manual_seed(100)
        x = torch.randn(world, 3, 5, 32)                  # what each rank has
        a, b = x.clone().requires_grad_(), x[rank].clone().requires_grad_()
        want, got = whole(a), part(b)
        assert torch.allclose(got, want[rank], atol=1e-5)
        want.square().sum().backward()
        got.square().sum().backward()
        assert torch.allclose(b.grad, a.grad[rank], atol=1e-4)
        for name in ("w1", "w2", "w3"):                   # the experts of this rank have seen the tokens of all
            assert torch.allclose(getattr(part.experts, name).grad, getattr(whole.experts, name).grad[mine], atol=1e-4)
        with open(os.path.join(result_dir, f"routed_ok_{rank}"), "w") as f:
            f.write("ok")
    except Exception:
        with open(os.path.join(result_dir, f"err_{rank}.txt"), "w") as f:
            f.write(traceback.format_exc())
        raise
    finally:
        dist.destroy_process_group()
