"""The training step of the smoke denoiser with more than 256 pixels per frame at the bottleneck (images of 128 x 128 and up in the production
net; here two levels, so 64 x 64 gives 1024): loss and every parameter gradient against autograd through the CPU oracle, at the tolerance of the
other training tests (1e-3 of a tensor's largest entry + 1e-4 of the net's largest gradient)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [48, 64])
def test_training_gradients_beyond_256_bottleneck_pixels(size):
    from diffphycon_amd.model.video_diffusion_pytorch.unet3d_train import TrainableUnet3D
    from diffphycon_amd.model.video_diffusion_pytorch.video_diffusion_pytorch_conv3d import Unet3D_with_Conv3D
    from oracle import train_smoke as TS
    from oracle import unet3d as O
    assert torch.cuda.is_available(), "GPU tests need a real MI355X"
    dev = torch.device("cuda:0")
    cfg = O.Unet3DConfig(dim=16, dim_mults=(1, 2), channels=6)
    sd = O.synthetic_state_dict(cfg, seed=3)
    m = Unet3D_with_Conv3D(dim=16, dim_mults=(1, 2), channels=6)
    m.load_state_dict(sd)
    T = TrainableUnet3D(m, dev)
    ts = TS.schedule(1000)
    g = torch.Generator().manual_seed(5)
    B, F = 1, 2
    x0, noise = (torch.randn(B, F, 6, size, size, generator=g) for _ in range(2))
    t = torch.tensor([300])
    want, grads = TS.loss_and_grads(sd, cfg, ts, x0 * 0.5, t, noise)
    loss = T.p_losses((x0 * 0.5).to(dev), t.to(dev), noise.to(dev), ts["sqrt_alphas_cumprod"].to(dev), ts["sqrt_one_minus_alphas_cumprod"].to(dev))
    assert abs(loss.item() - want.item()) < 1e-4 * want.item()
    G = max(v.abs().max().item() for v in grads.values())
    for k, v in grads.items():
        err = (T.ctx.G[k].cpu().reshape(v.shape) - v).abs().max().item()
        assert err < 1e-3 * (v.abs().max().item() + 1e-4 * G) + 1e-7 * G, (k, err, v.abs().max().item())
